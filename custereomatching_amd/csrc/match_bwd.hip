// Backward of the row matching operators (match.h).  Nothing of the forward's scores is kept: both kernels
// recompute them from q, k and the forward's log-sum-exp.
//   attention      P = exp(s - lse), dP = go . v, dS = P (dP - delta):  dq = S dS k,  dk = S dS^T q,  dv = P^T go
//   cross entropy  dS = w (P - [j = target])                           (HDV = 0)
// k_match_bwd_q owns query rows and walks the keys, k_match_bwd_k owns keys and walks the query rows: every
// result has one owner and one order of summation, no atomics.  The price is that scores (and dP) are
// computed twice.  dS and P are rounded to the inputs' 16 bits for their products (in two parts where kSplit says
// so), sums are in 32 bits.
//
// What bounds it: on 2048 rows of 1792 x 2048, 257 seen by each, 128 channels, dq takes 1.2 ms and dk 1.3 ms (2.6
// TB/s): matrix instructions 31 % of the time, the vector unit 42 %, two waves a SIMD that wait for LDS and, at a
// workgroup's start, for memory.  Three waves a SIMD spill; reading operands four ahead (as the forward does) spills
// in dk (1.8 ms) and changes nothing in dq.
#include <type_traits>

#include "match.h"
#include "match_launch.h"

namespace custma {
namespace {

template <int HD, int HDV>
struct BwdShape {
    static constexpr int KT = HD <= 128 ? 64 : 32;  // keys a tile (dq)
    static constexpr int RT = HD <= 128 ? 64 : 32;  // rows a tile (dk, dv)
    static constexpr int NKC = HD / 8, NVC = HDV / 8;
    static constexpr int kTileQ = KT * (HD + HDV) * 2;
    static constexpr int kLists = 3 * RT * 4, kTileK = RT * (HD + HDV) * 2 + kLists;
    // dS and P go into their products as two 16-bit parts where the values are narrow and for the cross entropy.  Their
    // rows sum to zero against keys that neighbouring columns nearly share, so a single rounding of each cost three
    // (float16) to eight (bfloat16) times the rounding of the result in dq and dk; two parts cost 9 % of the backward.
    // Wider values take the single rounding: on random heads of 64 channels dq, dk and dv are off by 2.4e-3 of their norm
    // (bfloat16) instead of the 1.65e-3 of the result's own rounding.
    static constexpr bool kSplit = HDV <= 32;
    // workgroups a compute unit that the registers are held to (three would spill: 1482 us against 1004 for dq of the
    // cross entropy on 2048 x 2048, D = 256, 128 channels)
    static constexpr int kWavesQ = HD <= 128 ? 2 : 1;
    static constexpr int kWavesK = HD <= 128 && HDV <= 64 ? 2 : 1;
    // buffers: as many as leave room for them, two to four
    static constexpr int stages(int tile) { return 4 * tile <= 79872 ? 4 : 3 * tile <= 79872 ? 3 : 2; }
    static constexpr int STQ = stages(kTileQ), STK = stages(kTileK);
    static constexpr int NLQ = fill_loads(KT, NKC, 4) + fill_loads(KT, NVC, 4);
    static constexpr int NLK = fill_loads(RT, NKC, 4) + fill_loads(RT, NVC, 4);
    static constexpr int kLdsQ = STQ * kTileQ, kLdsK = STK * kTileK;
};

// s += tile a's 32 rows times x, dp += tile b's times y; operands from LDS four at a time: their latency is paid once
template <typename E, int NKC, int NVC>
__device__ __forceinline__ void product(const char* a, const char* b, int row, int lane, const ix4* x, const ix4* y,
                                        fx16& s, fx16& dp) {
#pragma unroll
    for (int s0 = 0; s0 < NKC / 2; s0 += 4) {
        ix4 f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (s0 + i < NKC / 2) f[i] = frag_rows<NKC>(a, row, s0 + i, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (s0 + i < NKC / 2) s = Half16<E>::mma(f[i], x[s0 + i], s);
    }
    if constexpr (NVC > 0) {
#pragma unroll
        for (int s0 = 0; s0 < NVC / 2; s0 += 4) {
            ix4 f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (s0 + i < NVC / 2) f[i] = frag_rows<NVC>(b, row, s0 + i, lane);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (s0 + i < NVC / 2) dp = Half16<E>::mma(f[i], y[s0 + i], dp);
        }
    }
}

// what rounding (a, b) to `to` lost, rounded to 16 bits; CAREFUL: nothing where that is not finite
template <typename E, bool CAREFUL>
__device__ __forceinline__ int rest(int to, float a, float b) {
    const fx2 u = unpack2<E>(to);
    float x = a - u.x, y = b - u.y;
    if constexpr (CAREFUL) {
        x = fabsf(u.x) < INFINITY ? x : 0.f;
        y = fabsf(u.y) < INFINITY ? y : 0.f;
    }
    return pack2<E>(x, y);
}

template <typename E, int HD, int HDV>
__global__ __launch_bounds__(256, (BwdShape<HD, HDV>::kWavesQ)) void k_match_bwd_q(MatchGeo g, BwdArgs a, int row_tiles) {
    using S = BwdShape<HD, HDV>;
    typedef Half16<E> X;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = lane >> 5, col = lane & 31;
    uint32_t id = xcd_block();
    const int rt = (int)split_off(id, row_tiles), hk = (int)split_off(id, g.Hkv), b = (int)id;

    const int32_t off = first_position(g, b);
    const int32_t len = key_length(g, b), rows = g.rows();
    const int r0 = rt * 128, r = r0 + wave * 32 + col;
    const int last = r0 + 128 < rows ? r0 + 127 : rows - 1;
    const Span first_s = span_of(g, off, len, position_of_row(g, r0)), last_s = span_of(g, off, len, position_of_row(g, last));
    const bool live = r < rows;
    const int i = position_of_row(g, live ? r : rows - 1), gh = (live ? r : rows - 1) - i * g.G;
    Span me = span_of(g, off, len, i);
    if (!live) me.lo = me.hi = 0;
    const int mysink = me.hi < g.sinks ? me.hi : g.sinks;
    const int w0 = r0 + wave * 32;
    const bool wave_live = w0 < rows, wave_full = w0 + 31 < rows;
    const Span wf = span_of(g, off, len, position_of_row(g, wave_live ? w0 : rows - 1));
    const Span wl = span_of(g, off, len, position_of_row(g, wave_full ? w0 + 31 : rows - 1));

    int sink_end = g.sinks < first_s.lo ? g.sinks : first_s.lo;
    if (sink_end > last_s.hi) sink_end = last_s.hi;
    if (sink_end < 0) sink_end = 0;
    const int sink_tiles = (sink_end + S::KT - 1) / S::KT;
    const int win = last_s.hi > first_s.lo ? last_s.hi - first_s.lo : 0;
    const int tiles = sink_tiles + (win + S::KT - 1) / S::KT;

    const char* kb = (const char*)a.k + ((int64_t)b * g.ks[0] + (int64_t)hk * g.ks[2]) * 2;
    const char* vb = HDV ? (const char*)a.v + ((int64_t)b * g.vs[0] + (int64_t)hk * g.vs[2]) * 2 : nullptr;
    const int kchunks = g.C / 8, vchunks = g.Cv / 8;
    auto tile_range = [&](int t, int& ks, int& ke) {
        if (t < sink_tiles) {
            ks = t * S::KT;
            ke = sink_end;
        } else {
            ks = first_s.lo + (t - sink_tiles) * S::KT;
            ke = last_s.hi;
        }
    };
    const uint32_t lds0 = lds_offset(lds);
    const uint32_t kst = (uint32_t)(g.ks[1] * 2), vst = (uint32_t)(g.vs[1] * 2);
    Filler<S::KT, S::NKC, 4> kfill;
    Filler<S::KT, HDV ? S::NVC : 4, 4> vfill;
    kfill.init(kchunks, wave, lane, [&](int r) { return r * kst; });
    if constexpr (HDV > 0) vfill.init(vchunks, wave, lane, [&](int r) { return r * vst; });
    const int64_t kstep = (int64_t)S::KT * kst, vstep = (int64_t)S::KT * vst;
    auto seek = [&](KeyWalk& w, int t) __attribute__((always_inline)) {
        w.tile = t;
        tile_range(t, w.key, w.end);
        w.k = kb + (int64_t)w.key * kst;
        if constexpr (HDV > 0) w.v = vb + (int64_t)w.key * vst;
    };
    auto next = [&](KeyWalk& w, bool with_vectors) __attribute__((always_inline)) {
        ++w.tile;
        w.key += S::KT;
        if (with_vectors) {
            w.k += kstep;
            if constexpr (HDV > 0) w.v += vstep;
        }
        if (sink_tiles > 0 && w.tile == sink_tiles) seek(w, sink_tiles);
    };
    KeyWalk ahead;               // the next tile to fill
    uint32_t ahead_at;           // and its buffer
    auto fill = [&]() __attribute__((always_inline)) {
        kfill.fill(ahead_at, ahead.k, ahead.end - ahead.key, [&](int r) { return r * kst; });
        if constexpr (HDV > 0)
            vfill.fill(ahead_at + S::KT * HD * 2, ahead.v, ahead.end - ahead.key, [&](int r) { return r * vst; });
        next(ahead, true);
        ahead_at = ahead_at == lds0 + (S::STQ - 1) * S::kTileQ ? lds0 : ahead_at + S::kTileQ;
    };
#pragma unroll
    for (int x = 0; x < S::STQ; ++x) {
        clear_tails<S::NKC, 256>(lds + x * S::kTileQ, S::KT, kchunks);
        if constexpr (HDV > 0) clear_tails<S::NVC, 256>(lds + x * S::kTileQ + S::KT * HD * 2, S::KT, vchunks);
    }
    auto fill_first = [&]() __attribute__((always_inline)) {
        seek(ahead, 0);
        ahead_at = lds0;
#pragma unroll
        for (int x = 0; x < S::STQ - 1; ++x)
            if (0 + x < tiles) fill();
    };
    fill_first();

    const int64_t row = ((int64_t)b * g.Lq + i) * g.heads() + hk * g.G + gh;
    ix4 qf[HD / 16], gf[HDV ? HDV / 16 : 1];
    {
        const char* qr = (const char*)a.q + ((int64_t)b * g.qs[0] + (int64_t)i * g.qs[1] + (int64_t)(hk * g.G + gh) * g.qs[2]) * 2;
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) {
            const int c = 2 * s + h;
            qf[s] = c < kchunks ? *(const ix4*)(qr + c * 16) : ix4{0, 0, 0, 0};
        }
        if constexpr (HDV > 0) {
            const char* gr = (const char*)a.go + row * g.Cv * 2;
#pragma unroll
            for (int s = 0; s < HDV / 16; ++s) {
                const int c = 2 * s + h;
                gf[s] = c < vchunks ? *(const ix4*)(gr + c * 16) : ix4{0, 0, 0, 0};
            }
        }
    }
    const float sc = score_factor(g.scale);
#pragma unroll
    for (int s = 0; s < HD / 16; ++s) qf[s] = flip_sign(qf[s], g.scale);
    constexpr float kLift = HDV ? 0.f : X::kLift;
    const int64_t at = ((int64_t)b * g.Hkv + hk) * rows + (live ? r : rows - 1);
    const float begin = a.start[at] * sc, second = a.second[at];
    const int target = HDV == 0 && live ? a.hot[at] : -1;
    if constexpr (HDV == 0) {  // a row that does not count sees nothing
        if (second == 0.f) me.lo = me.hi = 0;
    }
    const float hot = __builtin_ldexpf(1.f, (int)kLift);
    fx16 acc[HD / 32];
    auto walk = [&](auto careful_c) __attribute__((always_inline)) {
        constexpr bool CAREFUL = decltype(careful_c)::value;
#pragma unroll
        for (int c = 0; c < HD / 32; ++c)
#pragma unroll
            for (int x = 0; x < 16; ++x) acc[c][x] = 0.f;
        KeyWalk now;
        seek(now, 0);
        int tile_at = 0;
        for (int t = 0; t < tiles; ++t, next(now, false), tile_at = tile_at == (S::STQ - 1) * S::kTileQ ? 0 : tile_at + S::kTileQ) {
            wait_tile<S::STQ, S::NLQ>(tiles - 1 - t);
            if (ahead.tile < tiles) fill();
            const int ks = now.key, ke = now.end;
            const bool sink_tile = t < sink_tiles;
            const char* kt = lds + tile_at;
            const char* vt = kt + S::KT * HD * 2;
#pragma unroll 1
            for (int u = 0; u < S::KT / 32; ++u) {
                const int k0 = ks + u * 32;
                if (!(wave_live && k0 < ke && (sink_tile || (k0 < wl.hi && (k0 + 32 > wf.lo || (g.sinks > 0 && k0 < g.sinks)))))) continue;
                const bool all = !sink_tile && wave_full && k0 >= wl.lo && k0 + 32 <= wf.hi;
                const int from = k0 + 4 * h, rel = from - me.lo, end = me.hi < ke ? me.hi : ke;
                const unsigned wide = (unsigned)(end - me.lo > 0 ? end - me.lo : 0);
                const bool sinks_here = g.sinks > 0 && k0 < g.sinks;
                fx16 s, dp;
#pragma unroll
                for (int x = 0; x < 16; ++x) s[x] = 0.f, dp[x] = second;
                product<E, S::NKC, S::NVC>(kt, vt, u * 32, lane, qf, gf, s, dp);
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const float p = exp2_hw(__builtin_fmaf(s[x], sc, begin));
                    s[x] = HDV > 0 ? p * dp[x] : p;
                }
                if constexpr (HDV == 0) {
                    if (__any(target >= k0 && target < k0 + 32)) {
                        const int tj = target - from;
#pragma unroll
                        for (int x = 0; x < 16; ++x)
                            if (tj == 8 * (x / 4) + x % 4) s[x] -= hot;
                    }
                }
                if (!all) {
                    if (sinks_here) {
#pragma unroll
                        for (int x = 0; x < 16; ++x) {
                            const int at = 8 * (x / 4) + x % 4;
                            const bool see = (unsigned)(rel + at) < wide || (from + at < mysink && from + at < ke);
                            s[x] = see ? s[x] : 0.f;
                        }
                    } else {
#pragma unroll
                        for (int x = 0; x < 16; ++x) s[x] = (unsigned)(rel + 8 * (x / 4) + x % 4) < wide ? s[x] : 0.f;
                    }
                }
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    ix4 df, dl;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float a0 = s[st * 8 + 2 * x], a1 = s[st * 8 + 2 * x + 1];
                        df[x] = pack2<E>(a0, a1);
                        if constexpr (S::kSplit) dl[x] = rest<E, CAREFUL>(df[x], a0, a1);
                    }
#pragma unroll
                    for (int c = 0; c < HD / 32; ++c) {
                        ix4 kc = frag_cols<S::NKC>(kt, u * 32 + st * 16, c * 32, lane);
                        // a key that is not finite has made its visible pairs' dS NaN already
                        if constexpr (CAREFUL) kc = all ? kc : finite_part<E>(kc);
                        acc[c] = X::mma(kc, df, acc[c]);
                        if constexpr (S::kSplit) acc[c] = X::mma(kc, dl, acc[c]);
                    }
                }
            }
        }
    };
    walk(std::false_type{});
    if (__syncthreads_or(any_not_finite(acc, 0.f))) {
        fill_first();
        walk(std::true_type{});
        __syncthreads();  // the tiles make room for the results
    }
    float f = g.scale * (a.factor ? a.factor[0] : 1.f) * (HDV == 0 ? second / hot : 1.f);
    if (HDV == 0 && second == 0.f) {  // weight 0 drops the row even where its scores are not finite
        f = 0.f;
#pragma unroll
        for (int c = 0; c < HD / 32; ++c)
#pragma unroll
            for (int x = 0; x < 16; ++x) acc[c][x] = 0.f;
    }
    static_assert(4 * 32 * HD * 2 <= S::kLdsQ, "the waves' rows fit where the tiles were");
    store_rows<E, S::NKC>(lds + wave * 32 * HD * 2, acc, f, g.C, lane, [&](int x) -> char* {
        const int rx = w0 + x;
        if (rx >= rows) return nullptr;
        const int ix = position_of_row(g, rx);
        return (char*)a.gq + ((((int64_t)b * g.Lq + ix) * g.Hkv + hk) * g.G + (rx - ix * g.G)) * g.C * 2;
    });
}

// Keys [kt * 128, + 128), 32 a wave.  SINKS: only the pairs of a sink key in front of its query's window;
// otherwise only the pairs inside windows (sinks in front of a window come in through init_k / init_v).
// GV: with the values' gradient; row matching on columns does not ask for it, and without it nothing spills (with it 60 to
// 72 bytes a lane at 128 / 32 channels and 700 to 780 at 256 / 256).
template <typename E, int HD, int HDV, bool SINKS, bool GV>
__global__ __launch_bounds__(256, (BwdShape<HD, HDV>::kWavesK)) void k_match_bwd_k(MatchGeo g, BwdArgs a, int key_tiles, int nsplit) {
    using S = BwdShape<HD, HDV>;
    typedef Half16<E> X;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = lane >> 5, col = lane & 31;
    uint32_t id = xcd_block();
    const int split = (int)split_off(id, nsplit), kt = (int)split_off(id, key_tiles);
    const int hk = (int)split_off(id, g.Hkv), b = (int)id;

    const int32_t off = first_position(g, b);
    const int32_t len = key_length(g, b), rows = g.rows();
    const int nkeys = SINKS ? (g.sinks < g.Lk ? g.sinks : g.Lk) : g.Lk;  // keys of the result
    const int k0 = kt * 128, kw = k0 + wave * 32, j = kw + col;
    const int kend = k0 + 128 < len ? k0 + 128 : len;  // behind the last key in use of this block
    // The rows that see a key are contiguous too, [row_lo(j), row_hi(j)), and both bounds ascend with the key.
    auto clamp_row = [&](int64_t i) { return i <= 0 ? 0 : i >= g.Lq ? rows : (int)i * g.G; };
    auto row_lo = [&](int key) {
        if (SINKS) return clamp_row((int64_t)key + g.left + 1 - off);  // key in front of the window
        return g.right < 0 ? 0 : clamp_row((int64_t)key - g.right - off);
    };
    auto row_hi = [&](int key) { return SINKS || g.left < 0 ? rows : clamp_row((int64_t)key + g.left + 1 - off); };
    const bool used = k0 < kend && (!SINKS || g.left >= 0);
    const int ra = used ? row_lo(k0) : 0, rb = used ? row_hi(kend - 1) : 0;
    const int tiles_all = rb > ra ? (rb - ra + S::RT - 1) / S::RT : 0;
    const int t0 = part_of(tiles_all, split, nsplit), t1 = part_of(tiles_all, split + 1, nsplit);
    const bool mine_used = used && j < kend;
    const int my_lo = mine_used ? row_lo(j) : 0, my_hi = mine_used ? row_hi(j) : 0;
    // rows that some key of the wave is seen by, and that all of them are
    const bool wave_used = used && kw < kend;
    const int wlast = kw + 31 < kend ? kw + 31 : kend - 1;
    const int some_lo = wave_used ? row_lo(kw) : 0, some_hi = wave_used ? row_hi(wlast) : 0;
    const int all_lo = wave_used ? row_lo(wlast) : 0, all_hi = wave_used && kw + 31 < kend ? row_hi(kw) : 0;

    const int kchunks = g.C / 8, vchunks = g.Cv / 8;
    const int64_t heads = g.heads();
    constexpr float kLift = HDV ? 0.f : X::kLift;
    const float hot = __builtin_ldexpf(1.f, (int)kLift);
    const float sc = score_factor(g.scale);
    const uint32_t lds0 = lds_offset(lds);
    const int64_t list = ((int64_t)b * g.Hkv + hk) * rows;  // of the rows' values
    const int64_t q_at = (int64_t)b * g.qs[0] + (int64_t)hk * g.G * g.qs[2];
    const int64_t go_at = (int64_t)b * g.Lq * heads + (int64_t)hk * g.G;
    // packed rows: where the group divides the tile, the rows of every tile lie alike
    const bool alike = S::RT % g.G == 0;
    auto q_off = [&](int x) {
        const int i = g.G == 1 ? x : x / g.G;
        return (uint32_t)(((int64_t)i * g.qs[1] + (int64_t)(x - i * g.G) * g.qs[2]) * 2);
    };
    auto go_off = [&](int x) {
        const int i = g.G == 1 ? x : x / g.G;
        return (uint32_t)(((int64_t)i * heads + (x - i * g.G)) * g.Cv * 2);
    };
    Filler<S::RT, S::NKC, 4> qfill;
    Filler<S::RT, HDV ? S::NVC : 4, 4> gfill;
    qfill.init(kchunks, wave, lane, q_off);
    if constexpr (HDV > 0) gfill.init(vchunks, wave, lane, go_off);
#pragma unroll
    for (int x = 0; x < S::STK; ++x) {
        clear_tails<S::NKC, 256>(lds + x * S::kTileK, S::RT, kchunks);
        if constexpr (HDV > 0) clear_tails<S::NVC, 256>(lds + x * S::kTileK + S::RT * HD * 2, S::RT, vchunks);
    }
    int ahead, ahead_row;           // the next tile to fill, its first row
    uint32_t ahead_at;              // its buffer
    const char *ahead_q, *ahead_go; // its first row's vectors (alike)
    const int per_tile = S::RT / g.G;
    auto seek = [&](int t) __attribute__((always_inline)) {
        ahead = t;
        ahead_row = ra + t * S::RT;
        const int i1 = position_of_row(g, ahead_row);
        ahead_q = (const char*)a.q + (q_at + (int64_t)i1 * g.qs[1]) * 2;
        if constexpr (HDV > 0) ahead_go = (const char*)a.go + (go_at + (int64_t)i1 * heads) * g.Cv * 2;
    };
    auto fill = [&]() __attribute__((always_inline)) {
        const uint32_t to = ahead_at;
        const int r1 = ahead_row;
        if (alike) {
            qfill.fill(to, ahead_q, rb - r1, q_off);
            if constexpr (HDV > 0) gfill.fill(to + S::RT * HD * 2, ahead_go, rb - r1, go_off);
        } else {
            fill_rows<S::RT, S::NKC, 4>(
                to,
                [&](int x) -> const char* {
                    const int r = r1 + x;
                    if (r >= rb) return nullptr;
                    const int i = r / g.G;
                    return (const char*)a.q + (q_at + (int64_t)i * g.qs[1] + (int64_t)(r - i * g.G) * g.qs[2]) * 2;
                },
                kchunks, wave, lane);
            if constexpr (HDV > 0)
                fill_rows<S::RT, S::NVC, 4>(
                    to + S::RT * HD * 2,
                    [&](int x) -> const char* {
                        const int r = r1 + x;
                        if (r >= rb) return nullptr;
                        const int i = r / g.G;
                        return (const char*)a.go + (go_at + (int64_t)i * heads + (r - i * g.G)) * g.Cv * 2;
                    },
                    vchunks, wave, lane);
        }
        // per row, one list a wave: what the score's product starts from, what dP's does (the weight), the target
        auto list_of = [&](const void* p, int n) {
            const int r = r1 + lane < rb ? r1 + lane : rb - 1;
            if (lane < S::RT) load_lds4((const char*)p + (list + r) * 4, to + S::RT * (HD + HDV) * 2 + n * S::RT * 4);
        };
        if (wave == 0) list_of(a.start, 0);
        else if (wave == 1) list_of(a.second, 1);
        else if (HDV == 0 && wave == 2) list_of(a.hot, 2);
        ++ahead;
        ahead_row += S::RT;
        ahead_q += (int64_t)per_tile * g.qs[1] * 2;
        if constexpr (HDV > 0) ahead_go += (int64_t)per_tile * heads * g.Cv * 2;
        ahead_at = ahead_at == lds0 + (S::STK - 1) * S::kTileK ? lds0 : ahead_at + S::kTileK;
    };
    auto fill_first = [&]() __attribute__((always_inline)) {
        seek(t0);
        ahead_at = lds0;
#pragma unroll
        for (int x = 0; x < S::STK - 1; ++x)
            if (t0 + x < t1) fill();
    };
    fill_first();

    ix4 kf[HD / 16], vf[HDV ? HDV / 16 : 1];
    {
        const bool ok = j < len;
        const char* kr = (const char*)a.k + ((int64_t)b * g.ks[0] + (int64_t)j * g.ks[1] + (int64_t)hk * g.ks[2]) * 2;
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) {
            const int c = 2 * s + h;
            kf[s] = ok && c < kchunks ? *(const ix4*)(kr + c * 16) : ix4{0, 0, 0, 0};
        }
        if constexpr (HDV > 0) {
            const char* vr = (const char*)a.v + ((int64_t)b * g.vs[0] + (int64_t)j * g.vs[1] + (int64_t)hk * g.vs[2]) * 2;
#pragma unroll
            for (int s = 0; s < HDV / 16; ++s) {
                const int c = 2 * s + h;
                vf[s] = ok && c < vchunks ? *(const ix4*)(vr + c * 16) : ix4{0, 0, 0, 0};
            }
        }
    }
#pragma unroll
    for (int s = 0; s < HD / 16; ++s) kf[s] = flip_sign(kf[s], g.scale);
    constexpr int NV = HDV ? HDV / 32 : 1;
    const bool want_v = GV && (a.gv || a.part_v);
    fx16 ak[HD / 32], av[NV];
    auto walk = [&](auto careful_c) __attribute__((always_inline)) {
        constexpr bool CAREFUL = decltype(careful_c)::value;
#pragma unroll
        for (int c = 0; c < HD / 32; ++c)
#pragma unroll
            for (int x = 0; x < 16; ++x) ak[c][x] = 0.f;
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
            for (int x = 0; x < 16; ++x) av[c][x] = 0.f;
        int tile_at = 0;
        for (int t = t0; t < t1; ++t, tile_at = tile_at == (S::STK - 1) * S::kTileK ? 0 : tile_at + S::kTileK) {
            wait_tile<S::STK, S::NLK>(t1 - 1 - t);
            if (ahead < t1) fill();
            const char* qt = lds + tile_at;
            const char* gt = qt + S::RT * HD * 2;
            const float* mt = (const float*)(qt + S::RT * (HD + HDV) * 2);
            const int* tgt = (const int*)mt + 2 * S::RT;
#pragma unroll 1
            for (int v = 0; v < S::RT / 32; ++v) {
                const int r1 = ra + t * S::RT + v * 32;
                if (r1 >= some_hi || r1 + 32 <= some_lo) continue;
                const bool all = r1 >= all_lo && r1 + 32 <= all_hi;
                // lane = key, register = row: a lane's rows are r1 + 4 h + 8 * (x / 4) + x % 4
                const int rel = r1 + 4 * h - my_lo;
                const unsigned wide = (unsigned)(my_hi - my_lo);
                auto sees = [&](int x) { return (unsigned)(rel + 8 * (x / 4) + x % 4) < wide; };
                auto rows4 = [&](int x) { return v * 32 + 2 * x + 4 * h; };  // four in a row in the lists
                fx16 s, dp;
#pragma unroll
                for (int x = 0; x < 16; x += 4) {
                    const float4 z4 = *(const float4*)(mt + rows4(x));
                    s[x] = z4.x, s[x + 1] = z4.y, s[x + 2] = z4.z, s[x + 3] = z4.w;
                    if constexpr (HDV > 0) {
                        const float4 d4 = *(const float4*)(mt + S::RT + rows4(x));
                        dp[x] = d4.x, dp[x + 1] = d4.y, dp[x + 2] = d4.z, dp[x + 3] = d4.w;
                    }
                }
                uint32_t counts = 0xffff;  // careful: rows that do not count start from -inf
                if constexpr (CAREFUL) {
                    counts = 0;
#pragma unroll
                    for (int x = 0; x < 16; ++x) counts |= (sees(x) && s[x] > -INFINITY ? 1u : 0u) << x;
                }
                if (!all) {
#pragma unroll
                    for (int x = 0; x < 16; ++x) s[x] = sees(x) ? s[x] : -INFINITY;
                }
                product<E, S::NKC, S::NVC>(qt, gt, v * 32, lane, kf, vf, s, dp);
                float p[16];
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    p[x] = exp2_hw(s[x] * sc);
                    if constexpr (HDV > 0) s[x] = p[x] * dp[x];
                }
                if constexpr (HDV == 0) {
                    const int tl = tgt[v * 32 + col];
                    if (__any(tl >= kw && tl < kw + 32)) {
#pragma unroll
                        for (int x = 0; x < 16; x += 4) {
                            const ix4 t4 = *(const ix4*)(tgt + rows4(x));
#pragma unroll
                            for (int y = 0; y < 4; ++y) p[x + y] -= t4[y] == j ? hot : 0.f;
                        }
                        if (r1 + 32 > rb) {  // a row repeated behind the last one has its target too
#pragma unroll
                            for (int x = 0; x < 16; ++x) p[x] = sees(x) ? p[x] : 0.f;
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 16; ++x) s[x] = p[x];
                    if (a.weight) {
#pragma unroll
                        for (int x = 0; x < 16; x += 4) {
                            const float4 d4 = *(const float4*)(mt + S::RT + rows4(x));
                            s[x] *= d4.x, s[x + 1] *= d4.y, s[x + 2] *= d4.z, s[x + 3] *= d4.w;
                        }
                    }
                }
                if (CAREFUL) {
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        p[x] = counts >> x & 1 ? p[x] : 0.f;
                        s[x] = counts >> x & 1 ? s[x] : 0.f;
                    }
                }
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    ix4 df, dl, pf, pl, see;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int y = st * 8 + 2 * x;
                        df[x] = pack2<E>(s[y], s[y + 1]);
                        if constexpr (S::kSplit) dl[x] = rest<E, CAREFUL>(df[x], s[y], s[y + 1]);
                        if constexpr (GV) pf[x] = pack2<E>(p[y], p[y + 1]);
                        if constexpr (GV && S::kSplit) pl[x] = rest<E, CAREFUL>(pf[x], p[y], p[y + 1]);
                        if constexpr (CAREFUL) see[x] = pack_ones<E>(counts >> y & 1, counts >> (y + 1) & 1);
                    }
#pragma unroll
                    for (int c = 0; c < HD / 32; ++c) {
                        ix4 qc = frag_cols<S::NKC>(qt, v * 32 + st * 16, c * 32, lane);
                        // a query that is not finite has made its visible pairs' dS NaN already
                        if constexpr (CAREFUL) qc = finite_part<E>(qc);
                        ak[c] = X::mma(qc, df, ak[c]);
                        if constexpr (S::kSplit) ak[c] = X::mma(qc, dl, ak[c]);
                    }
                    if constexpr (GV) {
                        if (want_v) {
#pragma unroll
                            for (int c = 0; c < HDV / 32; ++c) {
                                ix4 gc = frag_cols<S::NVC>(gt, v * 32 + st * 16, c * 32, lane);
                                if constexpr (CAREFUL) {
                                    add_not_finite<E>(av[c], gc, see);
                                    gc = finite_part<E>(gc);
                                }
                                av[c] = X::mma(gc, pf, av[c]);
                                if constexpr (S::kSplit) av[c] = X::mma(gc, pl, av[c]);
                            }
                        }
                    }
                }
            }
        }
    };
    walk(std::false_type{});
    if (__syncthreads_or(any_not_finite(ak, 0.f) || (GV && any_not_finite(av, 0.f)))) {
        fill_first();
        walk(std::true_type{});
        __syncthreads();  // the tiles make room for the results
    }
    const float f = a.factor ? a.factor[0] : 1.f;
    if (!SINKS && a.init_keys > kw && split == 0 && j < a.init_keys) {  // what the sinks' own pass found
        auto add = [&](fx16* acc, int n, const float* init, int C) __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < n; ++c)
#pragma unroll
                for (int x = 0; x < 16; x += 4) {
                    const int ch = c * 32 + 2 * x + 4 * h;
                    if (ch >= C) continue;
                    const float4 z = *(const float4*)(init + (((int64_t)b * a.init_keys + j) * g.Hkv + hk) * C + ch);
                    acc[c][x] += z.x, acc[c][x + 1] += z.y, acc[c][x + 2] += z.z, acc[c][x + 3] += z.w;
                }
        };
        if (a.gk || a.part_k) add(ak, HD / 32, a.init_k, g.C);
        if constexpr (GV) {
            if (want_v) add(av, HDV / 32, a.init_v, g.Cv);
        }
    }
    auto put_part = [&](const fx16* acc, int n, float* part, int C) __attribute__((always_inline)) {
        if (j >= nkeys) return;
#pragma unroll
        for (int c = 0; c < n; ++c)
#pragma unroll
            for (int x = 0; x < 16; x += 4) {
                const int ch = c * 32 + 2 * x + 4 * h;
                if (ch < C)
                    *(float4*)(part + ((((int64_t)split * g.B + b) * nkeys + j) * g.Hkv + hk) * C + ch) =
                        make_float4(acc[c][x], acc[c][x + 1], acc[c][x + 2], acc[c][x + 3]);
            }
    };
    static_assert(4 * 32 * HD * 2 <= S::kLdsK, "the waves' rows fit where the tiles were");
    auto row_of = [&](char* out, int C, int x) -> char* {
        return kw + x < g.Lk ? out + (((int64_t)b * g.Lk + kw + x) * g.Hkv + hk) * C * 2 : nullptr;
    };
    char* mine = lds + wave * 32 * HD * 2;
    if (a.part_k) {
        put_part(ak, HD / 32, a.part_k, g.C);
    } else if (a.gk) {
        store_rows<E, S::NKC>(mine, ak, g.scale * f / hot, g.C, lane, [&](int x) { return row_of((char*)a.gk, g.C, x); });
    }
    if constexpr (GV) {
        if (a.part_v) {
            put_part(av, HDV / 32, a.part_v, g.Cv);
        } else if (a.gv) {
            __builtin_amdgcn_wave_barrier();
            store_rows<E, S::NVC>(mine, av, f, g.Cv, lane, [&](int x) { return row_of((char*)a.gv, g.Cv, x); });
        }
    }
}

template <typename E, int HD, int HDV>
hipError_t go_q(const MatchGeo& g, const BwdArgs& a, hipStream_t s) {
    using S = BwdShape<HD, HDV>;
    const int row_tiles = (int)cdiv(g.rows(), 128);
    auto fn = k_match_bwd_q<E, HD, HDV>;
    static std::atomic<uint64_t> lds_done{0};
    hipError_t e = allow_lds((const void*)fn, S::kLdsQ, lds_done);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(fn, dim3((unsigned)((int64_t)row_tiles * g.Hkv * g.B)), dim3(256), S::kLdsQ, s, g, a, row_tiles);
    return hipGetLastError();
}
template <typename E, int HD, int HDV, bool SINKS, bool GV>
hipError_t go_k(const MatchGeo& g, const BwdArgs& a, int nsplit, hipStream_t s) {
    using S = BwdShape<HD, HDV>;
    const int key_tiles = (int)cdiv(SINKS && g.sinks < g.Lk ? g.sinks : g.Lk, 128);
    auto fn = k_match_bwd_k<E, HD, HDV, SINKS, GV>;
    static std::atomic<uint64_t> lds_done{0};
    hipError_t e = allow_lds((const void*)fn, S::kLdsK, lds_done);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(fn, dim3((unsigned)((int64_t)nsplit * key_tiles * g.Hkv * g.B)), dim3(256), S::kLdsK, s, g, a,
                       key_tiles, nsplit);
    return hipGetLastError();
}
template <int HD, int HDV>
hipError_t go_k_any(const MatchGeo& g, bool bf, const BwdArgs& a, bool sinks, int nsplit, hipStream_t s) {
    if constexpr (HDV > 0) {
        if (sinks) return bf ? go_k<__bf16, HD, HDV, true, true>(g, a, nsplit, s) : go_k<_Float16, HD, HDV, true, true>(g, a, nsplit, s);
    }
    if constexpr (HDV == 32) {  // values of a few channels: columns, which have no gradient
        if (!a.gv) return bf ? go_k<__bf16, HD, HDV, false, false>(g, a, nsplit, s) : go_k<_Float16, HD, HDV, false, false>(g, a, nsplit, s);
    }
    return bf ? go_k<__bf16, HD, HDV, false, HDV != 0>(g, a, nsplit, s) : go_k<_Float16, HD, HDV, false, HDV != 0>(g, a, nsplit, s);
}
}  // namespace

#define CUSTMA_CAT_(a, b) a##b
#define CUSTMA_CAT(a, b) CUSTMA_CAT_(a, b)
hipError_t CUSTMA_CAT(launch_match_bwd_q_, CUSTMA_MATCH_HD)(const MatchGeo& g, int dtype, int hdv, const BwdArgs& a,
                                                           hipStream_t s) {
    constexpr int HD = CUSTMA_MATCH_HD;
    const bool bf = dtype == CUSTMA_BF16;
    if (hdv == 0) return bf ? go_q<__bf16, HD, 0>(g, a, s) : go_q<_Float16, HD, 0>(g, a, s);
    if (hdv == HD) return bf ? go_q<__bf16, HD, HD>(g, a, s) : go_q<_Float16, HD, HD>(g, a, s);
    if (hdv == 32) return bf ? go_q<__bf16, HD, 32>(g, a, s) : go_q<_Float16, HD, 32>(g, a, s);
    return hipErrorInvalidValue;
}
hipError_t CUSTMA_CAT(launch_match_bwd_k_, CUSTMA_MATCH_HD)(const MatchGeo& g, int dtype, int hdv, const BwdArgs& a,
                                                           bool sinks, int nsplit, hipStream_t s) {
    constexpr int HD = CUSTMA_MATCH_HD;
    const bool bf = dtype == CUSTMA_BF16;
    if (hdv == 0) return go_k_any<HD, 0>(g, bf, a, sinks, nsplit, s);
    if (hdv == HD) return go_k_any<HD, HD>(g, bf, a, sinks, nsplit, s);
    if (hdv == 32) return go_k_any<HD, 32>(g, bf, a, sinks, nsplit, s);
    return hipErrorInvalidValue;
}

}  // namespace custma
