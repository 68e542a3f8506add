// Forward of the row matching operators (match.h): one pass over the keys with the running maximum and sum
// of the softmax.  One workgroup = 4 waves; a wave owns 32 packed query rows (WK = 1) or, where there are few
// rows, the waves split each key tile between them and join at the end (WK > 1).  The next one to three key
// tiles are in flight into LDS while the present one is used.
//
//   attention      o = sum_j p_j v_j / sum_j p_j, lse = log sum_j exp(s_j)       (template HDV > 0)
//   cross entropy  lse and the target's score only                              (HDV = 0)
//
// P is rounded to the inputs' 16 bits for the product with V (each p off by at most half a step, their sum
// is kept in 32 bits); where the output is 32-bit, or narrow and to be differentiated, it is split into two
// 16-bit parts, so that the product keeps 32-bit accuracy.  A wide 16-bit output takes the single rounding: it is then
// off by 2.0e-3 to 2.3e-3 of its norm (bfloat16) instead of the 1.65e-3 that its own rounding costs, where two parts took
// the prompt below from 88 to 110 us and the single token from 106 to 110.
//
// What bounds it, measured on this card (copy 4.7 TB/s, 16-bit product 1.4 PFLOP/s):
//   16 heads on 4, 8192 queries and keys, window 1024, 128 channels, bfloat16: 86 to 103 us by box and clock, 630 to 750
//     TFLOP/s.  Matrix instructions run 39 % of the time and the vector unit 50 % (exponentials, sums, rounding, the
//     keys' addresses), each wave mostly one after the other.  64 rows a wave, which halves the reads from LDS, took
//     130 us: one wave a SIMD leaves nothing to run beside the exponentials.  32 keys a tile: the same within the noise.
//   1792 queries, 2048 keys, 257 seen by each, 128 channels, 2048 rows: 750 us with values (2.8 TB/s), 640 us without;
//     the vector unit 61 %, and the first tiles' way from memory in workgroups of 12 tiles.
//   one query, 32 k keys, 4 sequences of 8 key heads: 100 us, 3.6 TB/s: the cache's way from memory.
#include <type_traits>

#include "match.h"
#include "match_launch.h"

namespace custma {
namespace {

template <int HD, int HDV, int WK>
struct FwdShape {
    static constexpr int WR = 4 / WK;                         // waves along rows
    static constexpr int BR = 32 * WR;                        // rows per workgroup
    // 64 keys a wave with wide values; 32 otherwise, where more registers would cost a wave a SIMD
    static constexpr int KW = (WK == 1 && HD <= 128) ? (HDV <= 32 ? 32 : 64) : 32;  // keys per wave and tile
    static constexpr int KT = KW * WK;
    static constexpr int NKC = HD / 8, NVC = HDV / 8;
    static constexpr int kTile = KT * (HD + HDV) * 2;         // bytes
    // buffers: as many as leave room for two workgroups a compute unit, two to four
    static constexpr int ST = 4 * kTile <= 79872 ? 4 : 3 * kTile <= 79872 ? 3 : 2;
    static constexpr int NL = fill_loads(KT, NKC, 4) + fill_loads(KT, NVC, 4);
    static constexpr int kJoin = WK > 1 ? 32 * WR * WK * 8 + (HDV ? 32 * WR * (WK - 1) * HDV * 4 : 4 * 32 * 4) : 0;
    // the result's rows pass through LDS on their way out, behind what the waves join in
    static constexpr int kOut = kJoin + WR * 32 * HDV * 2;
    static constexpr int kLds = ST * kTile > kOut ? ST * kTile : kOut;
    // waves a SIMD that registers are kept for: 256 channels, whose tiles leave room for two workgroups, spill at more.
    // With 256 value channels two spill as well (750 to 1080 bytes a lane), and the single token's four waves at 128 / 128
    // do (90 to 130): the spills are the compiler's own, the asm loads write no register.
    static constexpr int kWaves = HD == 256 ? 2 : HDV == 0 ? 4 : HDV == 32 ? 3 : 2;
};

// SPLIT: P in two 16-bit parts, for a 32-bit output, and for narrow values whose backward needs go . out to the same
// accuracy as its own products (match_bwd.hip)
template <typename E, int HD, int HDV, int WK, bool WIDE_OUT, bool SPLIT>
__global__ __launch_bounds__(256, (FwdShape<HD, HDV, WK>::kWaves)) void k_match_fwd(MatchGeo g, const char* __restrict__ q, const char* __restrict__ k,
                                                   const char* __restrict__ v, FwdOut o, int nsplit, int row_tiles) {
    using S = FwdShape<HD, HDV, WK>;
    typedef Half16<E> X;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = lane >> 5, col = lane & 31;
    const int wr = wave % S::WR, wk = wave / S::WR;

    // neighbouring workgroups share a key head's tiles: split fastest, then row tile, then head, then batch
    uint32_t id = xcd_block();
    const int split = (int)split_off(id, nsplit), rt = (int)split_off(id, row_tiles);
    const int hk = (int)split_off(id, g.Hkv), b = (int)id;

    const int32_t off = first_position(g, b);
    const int32_t len = key_length(g, b), rows = g.rows();
    const int r0 = rt * S::BR, r = r0 + wr * 32 + col;
    const int last = r0 + S::BR < rows ? r0 + S::BR - 1 : rows - 1;
    const Span first_s = span_of(g, off, len, position_of_row(g, r0)), last_s = span_of(g, off, len, position_of_row(g, last));
    const bool live = r < rows;
    const int i = position_of_row(g, live ? r : rows - 1), gh = (live ? r : rows - 1) - i * g.G;
    Span me = span_of(g, off, len, i);
    if (!live) me.lo = me.hi = 0;
    const int mysink = me.hi < g.sinks ? me.hi : g.sinks;
    // what the whole wave can see of the window: rows ascend, so do both bounds
    const int wlast = r0 + wr * 32 + 31 < rows ? r0 + wr * 32 + 31 : rows - 1;
    const bool wave_live = r0 + wr * 32 < rows;
    const Span wf = span_of(g, off, len, position_of_row(g, wave_live ? r0 + wr * 32 : rows - 1));
    const Span wl = span_of(g, off, len, position_of_row(g, wlast));
    const bool wave_full = r0 + wr * 32 + 31 < rows;

    // key tiles: sinks in front of the window, then the window
    int sink_end = g.sinks < first_s.lo ? g.sinks : first_s.lo;
    if (sink_end > last_s.hi) sink_end = last_s.hi;
    if (sink_end < 0) sink_end = 0;
    const int sink_tiles = (sink_end + S::KT - 1) / S::KT;
    const int win = last_s.hi > first_s.lo ? last_s.hi - first_s.lo : 0;
    const int tiles = sink_tiles + (win + S::KT - 1) / S::KT;
    const int t0 = part_of(tiles, split, nsplit), t1 = part_of(tiles, split + 1, nsplit);

    const char* kb = k + ((int64_t)b * g.ks[0] + (int64_t)hk * g.ks[2]) * 2;
    const char* vb = HDV ? v + ((int64_t)b * g.vs[0] + (int64_t)hk * g.vs[2]) * 2 : nullptr;
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
    // window tiles that this wave's rows reach into, [act0, act1), and that all of them see whole, [all0, all1)
    auto tile_up = [&](int key) { return key <= 0 ? 0 : (key + S::KT - 1) / S::KT; };
    const int mine = first_s.lo + wk * S::KW;  // this wave's first key of window tile 0
    int act0 = sink_tiles, act1 = sink_tiles, all0 = sink_tiles, all1 = sink_tiles;
    if (wave_live) {
        act0 += first_s.lo < g.sinks ? 0 : tile_up(wf.lo - S::KW + 1 - mine);
        act1 += tile_up(wl.hi - mine);
        all0 += tile_up(wl.lo - mine);
        const int room = wf.hi - S::KW - mine;
        all1 += wave_full && room >= 0 ? room / S::KT + 1 : 0;
    }
    const uint32_t lds0 = lds_offset(lds);
    const uint32_t kst = (uint32_t)(g.ks[1] * 2), vst = (uint32_t)(g.vs[1] * 2);
    Filler<S::KT, S::NKC, 4> kfill;
    Filler<S::KT, HDV ? S::NVC : 4, 4> vfill;
    kfill.init(kchunks, wave, lane, [&](int r) { return r * kst; });
    if constexpr (HDV > 0) vfill.init(vchunks, wave, lane, [&](int r) { return r * vst; });
    auto fill = [&](int t, int buf) __attribute__((always_inline)) {
        int ks, ke;
        tile_range(t, ks, ke);
        const uint32_t to = lds0 + buf * S::kTile;
        kfill.fill(to, kb + (int64_t)ks * g.ks[1] * 2, ke - ks, [&](int r) { return r * kst; });
        if constexpr (HDV > 0)
            vfill.fill(to + S::KT * HD * 2, vb + (int64_t)ks * g.vs[1] * 2, ke - ks, [&](int r) { return r * vst; });
    };
#pragma unroll
    for (int x = 0; x < S::ST; ++x) {
        clear_tails<S::NKC, 256>(lds + x * S::kTile, S::KT, kchunks);
        if constexpr (HDV > 0) clear_tails<S::NVC, 256>(lds + x * S::kTile + S::KT * HD * 2, S::KT, vchunks);
    }
    auto fill_first = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < S::ST - 1; ++x)
            if (t0 + x < t1) fill(t0 + x, x);
    };
    fill_first();

    // the wave's queries stay in registers: B operand, column = query
    ix4 qf[HD / 16];
    {
        const char* qr = q + ((int64_t)b * g.qs[0] + (int64_t)i * g.qs[1] + (int64_t)(hk * g.G + gh) * g.qs[2]) * 2;
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) {
            const int c = 2 * s + h;
            qf[s] = c < kchunks ? *(const ix4*)(qr + c * 16) : ix4{0, 0, 0, 0};
        }
    }
    const float sc = score_factor(g.scale);
#pragma unroll
    for (int s = 0; s < HD / 16; ++s) qf[s] = flip_sign(qf[s], g.scale);
    int target = -1;
    if constexpr (HDV == 0) {
        const int64_t tj = live ? o.target[(int64_t)b * g.Lq + i] : -1;
        if (tj >= me.lo && tj < me.hi) target = (int)tj;  // otherwise not a candidate: the row does not count
    }
    float m = -INFINITY, base = 0.f, l = 0.f, picked = 0.f;
    constexpr int NA = HDV ? HDV / 32 : 1, NU = S::KW / 32;
    fx16 acc[NA];

    // The softmax's reference m follows the running maximum only when that has grown by more than kSlack: p stays
    // below 2^kSlack, and most tiles need neither an exchange between the halves nor a rescaling of the sums.
    constexpr float kSlack = 8.f;
    auto walk = [&](auto careful_c) __attribute__((always_inline)) {
        constexpr bool CAREFUL = decltype(careful_c)::value;
        m = -INFINITY, base = 0.f, l = 0.f, picked = 0.f;
#pragma unroll
        for (int c = 0; c < NA; ++c)
#pragma unroll
            for (int x = 0; x < 16; ++x) acc[c][x] = 0.f;
        for (int t = t0, buf = 0; t < t1; ++t, buf = buf + 1 < S::ST ? buf + 1 : 0) {
            wait_tile<S::ST, S::NL>(t1 - 1 - t);
            if (t + S::ST - 1 < t1) fill(t + S::ST - 1, buf ? buf - 1 : S::ST - 1);
            int ks, ke;
            tile_range(t, ks, ke);
            ks += wk * S::KW;  // this wave's keys of the tile
            if (t < sink_tiles ? wave_live && ks < ke : t >= act0 && t < act1) {
                const char* kt = lds + buf * S::kTile;
                const char* vt = kt + S::KT * HD * 2;
                const bool all = t >= all0 && t < all1;
                fx16 s[NU];
                // a lane's keys are from + at, at = 8 * (x / 4) + x % 4: visible in [lo, hi) and below the sinks' end
                const int from = ks + 4 * h, lo = me.lo - from, hi = (me.hi < ke ? me.hi : ke) - from;
                const int sink = ks < g.sinks ? mysink - from : 0;
                const int rel = from - me.lo, end = me.hi < ke ? me.hi : ke;
                const unsigned wide = (unsigned)(end - me.lo > 0 ? end - me.lo : 0);
                const bool sinks_here = g.sinks > 0 && ks < g.sinks;
                auto sees = [&](int at) { return at < hi && (at >= lo || at < sink); };
#pragma unroll
                for (int u = 0; u < NU; ++u)
#pragma unroll
                    for (int x = 0; x < 16; ++x) s[u][x] = 0.f;
                // operands from LDS four at a time, the next four on their way while the present ones are multiplied
                constexpr int NF = HD / 16 * NU;
                ix4 kf[2][4];
                auto load = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
                    for (int y = 0; y < 4; ++y)
                        if (s0 + y < NF) kf[s0 / 4 % 2][y] = frag_rows<S::NKC>(kt, wk * S::KW + (s0 + y) % NU * 32, (s0 + y) / NU, lane);
                };
                load(0);
#pragma unroll
                for (int s0 = 0; s0 < NF; s0 += 4) {
                    load(s0 + 4);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int y = 0; y < 4; ++y)
                        if (s0 + y < NF) s[(s0 + y) % NU] = X::mma(kf[s0 / 4 % 2][y], qf[(s0 + y) / NU], s[(s0 + y) % NU]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (!all) {
                    // One path with 64 keys: where two meet, the compiler copies all scores on the way of whole tiles too
                    // (111 us instead of 103 for the prompt above).  With 32 it does not, and windows of a few tiles gain
                    // from the shorter test (2 to 3 % of the rows above).
                    if (NU == 1 && !sinks_here) {
#pragma unroll
                        for (int x = 0; x < 16; ++x) s[0][x] = (unsigned)(rel + 8 * (x / 4) + x % 4) < wide ? s[0][x] : -INFINITY;
                    } else {
#pragma unroll
                        for (int u = 0; u < NU; ++u)
#pragma unroll
                            for (int x = 0; x < 16; ++x) s[u][x] = sees(u * 32 + 8 * (x / 4) + x % 4) ? s[u][x] : -INFINITY;
                    }
                }
                float mt = -INFINITY;
#pragma unroll
                for (int u = 0; u < NU; ++u)
#pragma unroll
                    for (int x = 0; x < 16; x += 2) mt = fmaxf(fmaxf(s[u][x], s[u][x + 1]), mt);
                if constexpr (HDV == 0) {
                    if (__any(target >= ks && target < ks + S::KW)) {
                        const int tj = target - from;  // the target's place among this lane's scores
#pragma unroll
                        for (int u = 0; u < NU; ++u)
#pragma unroll
                            for (int x = 0; x < 16; ++x)
                                if (tj == u * 32 + 8 * (x / 4) + x % 4) picked = s[u][x] * sc;
                    }
                }
                if (__any(mt * sc > m + kSlack)) {
                    // only the rows that have grown: no row's rounding depends on the others of its wave
                    const float top = fmaxf(mt, other_half(mt)) * sc;
                    const float mn = top > m + kSlack ? top : m;
                    base = mn == -INFINITY ? 0.f : mn;
                    const float alpha = exp2_hw(m - base);
                    m = mn;
                    l *= alpha;
                    if constexpr (HDV > 0) {
#pragma unroll
                        for (int c = 0; c < NA; ++c)
#pragma unroll
                            for (int x = 0; x < 16; ++x) acc[c][x] *= alpha;
                    }
                }
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < NU; ++u)
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const float p = exp2_hw(__builtin_fmaf(s[u][x], sc, -base));
                        s[u][x] = p;
                        sum[x % 4] += p;
                    }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                if constexpr (HDV > 0) {
#pragma unroll
                    for (int u = 0; u < NU; ++u)
#pragma unroll
                        for (int st = 0; st < 2; ++st) {
                            ix4 pf, pl;
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                const float a = s[u][st * 8 + 2 * x], c = s[u][st * 8 + 2 * x + 1];
                                pf[x] = pack2<E>(a, c);
                                if constexpr (SPLIT) {
                                    const fx2 back = unpack2<E>(pf[x]);
                                    pl[x] = pack2<E>(a - back.x, c - back.y);
                                }
                            }
#pragma unroll
                            for (int c = 0; c < NA; ++c) {
                                ix4 vf = frag_cols<S::NVC>(vt, wk * S::KW + u * 32 + st * 16, c * 32, lane);
                                if constexpr (CAREFUL) {
                                    if (!all) {
                                        ix4 see;
#pragma unroll
                                        for (int x = 0; x < 4; ++x) {
                                            const int at = u * 32 + 16 * st + 8 * (x / 2) + 2 * (x % 2);
                                            see[x] = pack_ones<E>(sees(at), sees(at + 1));
                                        }
                                        add_not_finite<E>(acc[c], vf, see);
                                        vf = finite_part<E>(vf);
                                    }
                                }
                                acc[c] = X::mma(vf, pf, acc[c]);
                                if constexpr (SPLIT) acc[c] = X::mma(vf, pl, acc[c]);
                            }
                        }
                }
            }
        }
    };
    walk(std::false_type{});
    if constexpr (HDV > 0) {
        if (__syncthreads_or(any_not_finite(acc, l))) {
            fill_first();
            walk(std::true_type{});
            __syncthreads();  // the tiles make room for the results
        }
    } else {
        __syncthreads();
    }
    l += other_half(l);
    if constexpr (HDV == 0) {
        // exactly one of the wave's halves held the target's score, if any; the other's is 0
        picked += other_half(picked);
    }

    if constexpr (WK > 1) {  // join the waves that split the keys
        float* ml = (float*)lds;                   // [WK][BR][2]
        float* part = ml + 2 * S::BR * WK;         // [WK - 1][BR][HDV] or picked [WK][BR]
        if (h == 0) {
            ml[(wk * S::BR + wr * 32 + col) * 2] = m;
            ml[(wk * S::BR + wr * 32 + col) * 2 + 1] = l;
            if constexpr (HDV == 0) part[wk * S::BR + wr * 32 + col] = picked;
        }
        if constexpr (HDV > 0) {
            if (wk > 0) {
#pragma unroll
                for (int c = 0; c < HDV / 32; ++c)
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const int ch = c * 32 + 8 * (x / 4) + 4 * h + x % 4;
                        part[((wk - 1) * HDV + ch) * S::BR + wr * 32 + col] = acc[c][x];
                    }
            }
        }
        __syncthreads();
        if (wk > 0) return;
        float M = m;
#pragma unroll
        for (int w = 1; w < WK; ++w) M = fmaxf(M, ml[(w * S::BR + wr * 32 + col) * 2]);
        const float base = M == -INFINITY ? 0.f : M;
        float f = exp2_hw(m - base);
        l *= f;
        if constexpr (HDV > 0) {
#pragma unroll
            for (int c = 0; c < HDV / 32; ++c)
#pragma unroll
                for (int x = 0; x < 16; ++x) acc[c][x] *= f;
        }
#pragma unroll
        for (int w = 1; w < WK; ++w) {
            const float fw = exp2_hw(ml[(w * S::BR + wr * 32 + col) * 2] - base);
            l = __builtin_fmaf(fw, ml[(w * S::BR + wr * 32 + col) * 2 + 1], l);
            if constexpr (HDV > 0) {
#pragma unroll
                for (int c = 0; c < HDV / 32; ++c)
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const int ch = c * 32 + 8 * (x / 4) + 4 * h + x % 4;
                        acc[c][x] = __builtin_fmaf(fw, part[((w - 1) * HDV + ch) * S::BR + wr * 32 + col], acc[c][x]);
                    }
            } else {
                picked += part[w * S::BR + wr * 32 + col];
            }
        }
        m = M;
    }

    const int64_t row = ((int64_t)b * g.Lq + i) * g.heads() + hk * g.G + gh;
    if (nsplit > 1) {
        if (!live) return;
        const int64_t all = (int64_t)g.B * g.Lq * g.heads();
        if (h == 0) {
            float* to = o.part_ml + ((int64_t)split * all + row) * 4;
            to[0] = m;
            to[1] = l;
            to[2] = picked;
        }
        if constexpr (HDV > 0) {
            float* to = o.part + ((int64_t)split * all + row) * g.Cv;
#pragma unroll
            for (int c = 0; c < HDV / 32; ++c)
#pragma unroll
                for (int x = 0; x < 16; x += 4) {
                    const int ch = c * 32 + 2 * x + 4 * h;
                    if (ch < g.Cv) *(float4*)(to + ch) = make_float4(acc[c][x], acc[c][x + 1], acc[c][x + 2], acc[c][x + 3]);
                }
        }
        return;
    }
    const float lse = l == 0.f ? -INFINITY : (m + __builtin_log2f(l)) * kLn2;
    if constexpr (HDV == 0) {
        if (h == 0 && live) {
            o.lse[row] = lse;
            o.loss[row] = target >= 0 ? (m - picked + __builtin_log2f(l)) * kLn2 : 0.f;
        }
    } else {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (h == 0 && live && o.lse) o.lse[row] = lse;
        if constexpr (WIDE_OUT) {
            if (!live) return;
#pragma unroll
            for (int c = 0; c < HDV / 32; ++c)
#pragma unroll
                for (int x = 0; x < 16; x += 4) {
                    const int ch = c * 32 + 2 * x + 4 * h;
                    if (ch < g.Cv)
                        *(float4*)((float*)o.out + row * g.Cv + ch) = make_float4(acc[c][x] * inv, acc[c][x + 1] * inv,
                                                                                  acc[c][x + 2] * inv, acc[c][x + 3] * inv);
                }
        } else {
            char* mine_out = lds + S::kJoin + wr * 32 * HDV * 2;
            auto row_of = [&](void* base, int x) -> char* {
                const int rx = r0 + wr * 32 + x;
                if (rx >= rows) return nullptr;
                const int ix = position_of_row(g, rx);
                return (char*)base + ((((int64_t)b * g.Lq + ix) * g.Hkv + hk) * g.G + (rx - ix * g.G)) * g.Cv * 2;
            };
            store_rows<E, S::NVC>(mine_out, acc, inv, g.Cv, lane, [&](int x) { return row_of(o.out, x); });
            if (o.low) {
#pragma unroll
                for (int c = 0; c < HDV / 32; ++c)
#pragma unroll
                    for (int x = 0; x < 16; x += 2) {
                        const float a0 = acc[c][x] * inv, a1 = acc[c][x + 1] * inv;
                        const fx2 u = unpack2<E>(pack2<E>(a0, a1));
                        acc[c][x] = a0 - u.x;
                        acc[c][x + 1] = a1 - u.y;
                    }
                __builtin_amdgcn_wave_barrier();
                store_rows<E, S::NVC>(mine_out, acc, 1.f, g.Cv, lane, [&](int x) { return row_of(o.low, x); });
            }
        }
    }
}

template <typename E, int HD, int HDV, int WK, bool WIDE_OUT, bool SPLIT>
hipError_t launch_shape(const MatchGeo& g, const void* q, const void* k, const void* v, const FwdOut& o, int nsplit,
                        hipStream_t s) {
    using S = FwdShape<HD, HDV, WK>;
    const int row_tiles = (int)cdiv(g.rows(), S::BR);
    const int64_t blocks = (int64_t)nsplit * row_tiles * g.Hkv * g.B;
    auto fn = k_match_fwd<E, HD, HDV, WK, WIDE_OUT, SPLIT>;
    static std::atomic<uint64_t> lds_done{0};
    hipError_t e = allow_lds((const void*)fn, S::kLds, lds_done);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(256), S::kLds, s, g, (const char*)q, (const char*)k,
                       (const char*)v, o, nsplit, row_tiles);
    return hipGetLastError();
}

template <int HD, int HDV, int WK>
hipError_t launch_rows(const MatchGeo& g, bool bf, bool wide_out, const void* q, const void* k, const void* v, const FwdOut& o,
                       int nsplit, hipStream_t s) {
#define CUSTMA_GO(W, P) \
    return bf ? launch_shape<__bf16, HD, HDV, WK, W, P>(g, q, k, v, o, nsplit, s) : launch_shape<_Float16, HD, HDV, WK, W, P>(g, q, k, v, o, nsplit, s)
    if constexpr (HDV > 0) {
        if (wide_out) CUSTMA_GO(true, true);
    }
    if constexpr (HDV == 32) {
        if (o.low) CUSTMA_GO(false, true);
    }
    CUSTMA_GO(false, false);
#undef CUSTMA_GO
}
template <int HD, int HDV>
hipError_t launch_hd(const MatchGeo& g, bool bf, bool wide_out, bool few, const void* q, const void* k, const void* v,
                     const FwdOut& o, int nsplit, hipStream_t s) {
    if (few) return launch_rows<HD, HDV, HD == 256 ? 2 : 4>(g, bf, wide_out, q, k, v, o, nsplit, s);
    return launch_rows<HD, HDV, 1>(g, bf, wide_out, q, k, v, o, nsplit, s);
}
}  // namespace

#define CUSTMA_CAT_(a, b) a##b
#define CUSTMA_CAT(a, b) CUSTMA_CAT_(a, b)
// one translation unit per channel count: -DCUSTMA_MATCH_HD=32/64/128/256
hipError_t CUSTMA_CAT(launch_match_fwd_, CUSTMA_MATCH_HD)(const MatchGeo& g, int dtype, bool wide_out, bool few, int hdv,
                                                         const void* q, const void* k, const void* v, const FwdOut& o,
                                                         int nsplit, hipStream_t s) {
    constexpr int HD = CUSTMA_MATCH_HD;
    const bool bf = dtype == CUSTMA_BF16;
    if (hdv == 0) return launch_hd<HD, 0>(g, bf, wide_out, few, q, k, v, o, nsplit, s);
    if (hdv == HD) return launch_hd<HD, HD>(g, bf, wide_out, few, q, k, v, o, nsplit, s);
    if (HD > 32 && hdv == 32) return launch_hd<HD, 32>(g, bf, wide_out, few, q, k, v, o, nsplit, s);
    return hipErrorInvalidValue;
}

}  // namespace custma
