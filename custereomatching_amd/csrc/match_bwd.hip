// Backward of the row matching operators (match.h).  Nothing of the forward's scores is kept: both kernels
// recompute them from q, k and the forward's log-sum-exp.
//   attention      P = exp(s - lse), dP = go . v, dS = P (dP - delta):  dq = S dS k,  dk = S dS^T q,  dv = P^T go
//   cross entropy  dS = w (P - [j = target])                           (HDV = 0)
// k_match_bwd_q owns query rows and walks the keys, k_match_bwd_k owns keys and walks the query rows: every
// result has one owner and one order of summation, no atomics.  The price is that scores (and dP) are
// computed twice.  dS and P are rounded to the inputs' 16 bits for their products, sums are in 32 bits.
#include "match.h"
#include "match_launch.h"

namespace custma {
namespace {

template <int HD, int HDV>
struct BwdShape {
    static constexpr int KT = HD <= 128 ? 64 : 32;  // keys a tile (dq)
    static constexpr int RT = HD <= 128 ? 64 : 32;  // rows a tile (dk, dv)
    static constexpr int NKC = HD / 8, NVC = HDV / 8;
    static constexpr int kTileQ = KT * (HD + HDV) * 2, kLdsQ = 2 * kTileQ;
    static constexpr int kMeta = RT * 20, kTileK = RT * (HD + HDV) * 2 + kMeta, kLdsK = 2 * kTileK;
};

template <typename E, int HD, int HDV>
__global__ __launch_bounds__(256) void k_match_bwd_q(MatchGeo g, BwdArgs a, int row_tiles) {
    using S = BwdShape<HD, HDV>;
    typedef Half16<E> X;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = lane >> 5, col = lane & 31;
    int64_t id = xcd_remap(blockIdx.x, gridDim.x);
    const int rt = (int)(id % row_tiles);
    id /= row_tiles;
    const int hk = (int)(id % g.Hkv), b = (int)(id / g.Hkv);

    const int64_t off = g.offset ? g.offset[b] : 0;
    const int32_t len = key_length(g, b), rows = g.rows();
    const int r0 = rt * 128, r = r0 + wave * 32 + col;
    const int last = r0 + 128 < rows ? r0 + 127 : rows - 1;
    const Span first_s = span_of(g, off, len, r0 / g.G), last_s = span_of(g, off, len, last / g.G);
    const bool live = r < rows;
    const int i = (live ? r : rows - 1) / g.G, gh = (live ? r : rows - 1) % g.G;
    Span me = span_of(g, off, len, i);
    if (!live) me.lo = me.hi = 0;
    const int mysink = me.hi < g.sinks ? me.hi : g.sinks;
    const int w0 = r0 + wave * 32;
    const bool wave_live = w0 < rows, wave_full = w0 + 31 < rows;
    const Span wf = span_of(g, off, len, (wave_live ? w0 : rows - 1) / g.G);
    const Span wl = span_of(g, off, len, (wave_full ? w0 + 31 : rows - 1) / g.G);

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
    auto fill = [&](int t, int buf) {
        int ks, ke;
        tile_range(t, ks, ke);
        char* to = lds + buf * S::kTileQ;
        fill_tile<S::KT, S::NKC, 4>(to, kb, g.ks[1] * 2, ks, ke, kchunks, wave, lane);
        if constexpr (HDV > 0)
            fill_tile<S::KT, S::NVC, 4>(to + S::KT * HD * 2, vb, g.vs[1] * 2, ks, ke, vchunks, wave, lane);
    };
    if (tiles) fill(0, 0);

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
    const float sc = g.scale * kLog2e;
    constexpr float kLift = HDV ? 0.f : X::kLift;
    const float lse = a.lse[row];
    const float base = lse * kLog2e - kLift;
    const float delta = HDV ? a.delta[row] : 0.f;
    int target = -1;
    float weight = 1.f;
    if constexpr (HDV == 0) {
        const int64_t t = a.target[row];
        weight = live && t >= me.lo && t < me.hi ? (a.weight ? a.weight[row] : 1.f) : 0.f;
        target = t >= me.lo && t < me.hi ? (int)t : -1;
    }
    const float hot = __builtin_ldexpf(1.f, (int)kLift);
    fx16 acc[HD / 32];
#pragma unroll
    for (int c = 0; c < HD / 32; ++c)
#pragma unroll
        for (int t = 0; t < 16; ++t) acc[c][t] = 0.f;

    wait_fills();
    __syncthreads();
    for (int t = 0; t < tiles; ++t) {
        const int buf = t & 1;
        if (t + 1 < tiles) fill(t + 1, buf ^ 1);
        int ks, ke;
        tile_range(t, ks, ke);
        const bool sink_tile = t < sink_tiles;
        const char* kt = lds + buf * S::kTileQ;
        const char* vt = kt + S::KT * HD * 2;
#pragma unroll 1
        for (int u = 0; u < S::KT / 32; ++u) {
            const int k0 = ks + u * 32;
            if (!(wave_live && k0 < ke && (sink_tile || (k0 < wl.hi && (k0 + 32 > wf.lo || k0 < g.sinks))))) continue;
            fx16 s, dp;
#pragma unroll
            for (int x = 0; x < 16; ++x) s[x] = dp[x] = 0.f;
#pragma unroll
            for (int st = 0; st < HD / 16; ++st) s = X::mma(frag_rows<S::NKC>(kt, u * 32, st, lane), qf[st], s);
            if constexpr (HDV > 0) {
#pragma unroll
                for (int st = 0; st < HDV / 16; ++st) dp = X::mma(frag_rows<S::NVC>(vt, u * 32, st, lane), gf[st], dp);
            }
            const bool all = !sink_tile && wave_full && k0 >= wl.lo && k0 + 32 <= wf.hi;
            const int tj = target - k0 - 4 * h;
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const int at = 8 * (x / 4) + x % 4;
                float p = exp2_hw(__builtin_fmaf(s[x], sc, -base));
                float d;
                if constexpr (HDV > 0) d = p * (dp[x] - delta);
                else d = tj == at ? p - hot : p;
                if (!all) {
                    const int j = k0 + 4 * h + at;
                    const bool see = j < ke && j < me.hi && (j >= me.lo || j < mysink);
                    d = see ? d : 0.f;
                }
                s[x] = d;
            }
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                ix4 df;
#pragma unroll
                for (int x = 0; x < 4; ++x) df[x] = pack2<E>(s[st * 8 + 2 * x], s[st * 8 + 2 * x + 1]);
#pragma unroll
                for (int c = 0; c < HD / 32; ++c)
                    acc[c] = X::mma(frag_cols<S::NKC>(kt, u * 32 + st * 16, c * 32, lane), df, acc[c]);
            }
        }
        wait_fills();
        __syncthreads();
    }
    if (!live) return;
    // weight 0 drops the row even where its scores are not finite
    const float f = g.scale * (a.factor ? a.factor[0] : 1.f) * weight / hot;
    const bool none = HDV == 0 && weight == 0.f;
    char* to = (char*)a.gq + row * g.C * 2;
#pragma unroll
    for (int c = 0; c < HD / 32; ++c)
#pragma unroll
        for (int x = 0; x < 16; x += 4) {
            const int ch = c * 32 + 2 * x + 4 * h;
            if (ch >= g.C) continue;
            float o[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) o[y] = none ? 0.f : acc[c][x + y] * f;
            *(ix2*)(to + ch * 2) = ix2{pack2<E>(o[0], o[1]), pack2<E>(o[2], o[3])};
        }
}

// Keys [kt * 128, + 128), 32 a wave.  SINKS: only the pairs of a sink key in front of its query's window;
// otherwise only the pairs inside windows (sinks in front of a window come in through init_k / init_v).
template <typename E, int HD, int HDV, bool SINKS>
__global__ __launch_bounds__(256) void k_match_bwd_k(MatchGeo g, BwdArgs a, int key_tiles, int nsplit) {
    using S = BwdShape<HD, HDV>;
    typedef Half16<E> X;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = lane >> 5, col = lane & 31;
    int64_t id = xcd_remap(blockIdx.x, gridDim.x);
    const int split = (int)(id % nsplit);
    id /= nsplit;
    const int kt = (int)(id % key_tiles);
    id /= key_tiles;
    const int hk = (int)(id % g.Hkv), b = (int)(id / g.Hkv);

    const int64_t off = g.offset ? g.offset[b] : 0;
    const int32_t len = key_length(g, b);
    const int nkeys = SINKS ? (g.sinks < g.Lk ? g.sinks : g.Lk) : g.Lk;  // keys of the result
    const int k0 = kt * 128, kw = k0 + wave * 32, j = kw + col;
    const int kend = k0 + 128 < len ? k0 + 128 : len;  // last key in use of this block
    // query positions that can see a key of the block
    int64_t i0 = 0, i1 = g.Lq;
    if (SINKS) {
        if (g.left >= 0 && g.left + 1 - off > i0) i0 = g.left + 1 - off;
        if (g.left < 0) i1 = 0;
        if (g.right >= 0 && k0 - (int64_t)g.right - off > i0) i0 = k0 - (int64_t)g.right - off;
    } else {
        if (g.right >= 0 && k0 - (int64_t)g.right - off > i0) i0 = k0 - (int64_t)g.right - off;
        if (g.left >= 0 && kend + (int64_t)g.left - off < i1) i1 = kend + (int64_t)g.left - off;
    }
    if (k0 >= len || i1 < i0) i1 = i0 = 0;
    const int ra = (int)i0 * g.G, rb = (int)i1 * g.G;
    const int tiles_all = (rb - ra + S::RT - 1) / S::RT;
    const int t0 = (int)((int64_t)tiles_all * split / nsplit), t1 = (int)((int64_t)tiles_all * (split + 1) / nsplit);

    const int kchunks = g.C / 8, vchunks = g.Cv / 8;
    const int64_t heads = g.heads();
    auto row_id = [&](int r) { return ((int64_t)b * g.Lq + r / g.G) * heads + hk * g.G + r % g.G; };
    auto fill = [&](int t, int buf) {
        char* to = lds + buf * S::kTileK;
        const int r1 = ra + t * S::RT;
        fill_rows<S::RT, S::NKC, 4>(
            to,
            [&](int x) -> const char* {
                const int r = r1 + x;
                if (r >= rb) return nullptr;
                return (const char*)a.q + ((int64_t)b * g.qs[0] + (int64_t)(r / g.G) * g.qs[1] + (int64_t)(hk * g.G + r % g.G) * g.qs[2]) * 2;
            },
            kchunks, wave, lane);
        if constexpr (HDV > 0)
            fill_rows<S::RT, S::NVC, 4>(
                to + S::RT * HD * 2,
                [&](int x) -> const char* {
                    return r1 + x < rb ? (const char*)a.go + row_id(r1 + x) * g.Cv * 2 : nullptr;
                },
                vchunks, wave, lane);
    };
    // per row of a tile: log-sum-exp in base 2, delta or weight, visible keys [from, to), target
    constexpr float kLift = HDV ? 0.f : X::kLift;
    const float hot = __builtin_ldexpf(1.f, (int)kLift);
    auto meta = [&](int t, int buf) {
        const int x = threadIdx.x;
        if (x >= S::RT) return;
        float* to = (float*)(lds + buf * S::kTileK + S::RT * (HD + HDV) * 2);
        const int r = ra + t * S::RT + x;
        float lse = 0.f, d = 0.f;
        int from = 0, end = 0, target = -1;
        if (r < rb) {
            const int64_t row = row_id(r);
            const Span s = span_of(g, off, len, r / g.G);
            lse = a.lse[row] * kLog2e - kLift;
            if constexpr (HDV > 0) {
                d = a.delta[row];
            } else {
                const int64_t tj = a.target[row];
                const bool counts = tj >= s.lo && tj < s.hi;
                d = counts ? (a.weight ? a.weight[row] : 1.f) : 0.f;
                target = counts ? (int)tj : -1;
            }
            if (SINKS) {
                end = s.lo < g.sinks ? s.lo : g.sinks;
            } else {
                from = s.lo;
                end = s.hi;
            }
            if (HDV == 0 && d == 0.f) from = end = 0;  // a row that does not count
        }
        to[x] = lse;
        to[S::RT + x] = d;
        ((int*)to)[2 * S::RT + x] = from;
        ((int*)to)[3 * S::RT + x] = end;
        ((int*)to)[4 * S::RT + x] = target;
    };
    if (t0 < t1) {
        fill(t0, 0);
        meta(t0, 0);
    }

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
    const float sc = g.scale * kLog2e;
    fx16 ak[HD / 32], av[HDV ? HDV / 32 : 1];
#pragma unroll
    for (int c = 0; c < HD / 32; ++c)
#pragma unroll
        for (int x = 0; x < 16; ++x) ak[c][x] = 0.f;
#pragma unroll
    for (int c = 0; c < (HDV ? HDV / 32 : 1); ++c)
#pragma unroll
        for (int x = 0; x < 16; ++x) av[c][x] = 0.f;

    wait_fills();
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1;
        if (t + 1 < t1) {
            fill(t + 1, buf ^ 1);
            meta(t + 1, buf ^ 1);
        }
        const char* qt = lds + buf * S::kTileK;
        const char* gt = qt + S::RT * HD * 2;
        const float* mt = (const float*)(qt + S::RT * (HD + HDV) * 2);
        const int* from = (const int*)mt + 2 * S::RT;
        const int* end = from + S::RT;
        const int* tgt = end + S::RT;
#pragma unroll 1
        for (int u = 0; u < S::RT / 32; ++u) {
            // which of the 32 rows see which of the wave's 32 keys: by ballot over the rows' bounds
            const int fr = from[u * 32 + col], en = end[u * 32 + col];
            if (!__any(fr < kw + 32 && en > kw)) continue;
            const bool all = __all(fr <= kw && en >= kw + 32);
            fx16 s, dp;
#pragma unroll
            for (int x = 0; x < 16; ++x) s[x] = dp[x] = 0.f;
#pragma unroll
            for (int st = 0; st < HD / 16; ++st) s = X::mma(frag_rows<S::NKC>(qt, u * 32, st, lane), kf[st], s);
            if constexpr (HDV > 0) {
#pragma unroll
                for (int st = 0; st < HDV / 16; ++st) dp = X::mma(frag_rows<S::NVC>(gt, u * 32, st, lane), vf[st], dp);
            }
            float p[16];
#pragma unroll
            for (int x = 0; x < 16; x += 4) {
                const int at = u * 32 + 2 * x + 4 * h;
                const float4 lse = *(const float4*)(mt + at), d4 = *(const float4*)(mt + S::RT + at);
                int4 f4, e4, t4;
                if (!all) {
                    f4 = *(const int4*)(from + at);
                    e4 = *(const int4*)(end + at);
                }
                if constexpr (HDV == 0) t4 = *(const int4*)(tgt + at);
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const float ls = y == 0 ? lse.x : y == 1 ? lse.y : y == 2 ? lse.z : lse.w;
                    const float dd = y == 0 ? d4.x : y == 1 ? d4.y : y == 2 ? d4.z : d4.w;
                    float e = exp2_hw(__builtin_fmaf(s[x + y], sc, -ls)), d;
                    if constexpr (HDV > 0) {
                        d = e * (dp[x + y] - dd);
                    } else {
                        const int tj = y == 0 ? t4.x : y == 1 ? t4.y : y == 2 ? t4.z : t4.w;
                        d = dd * (tj == j ? e - hot : e);
                    }
                    if (!all) {
                        const int fj = y == 0 ? f4.x : y == 1 ? f4.y : y == 2 ? f4.z : f4.w;
                        const int ej = y == 0 ? e4.x : y == 1 ? e4.y : y == 2 ? e4.z : e4.w;
                        const bool see = j >= fj && j < ej;
                        e = see ? e : 0.f;
                        d = see ? d : 0.f;
                    }
                    p[x + y] = e;
                    s[x + y] = d;
                }
            }
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                ix4 df, pf;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    df[x] = pack2<E>(s[st * 8 + 2 * x], s[st * 8 + 2 * x + 1]);
                    pf[x] = pack2<E>(p[st * 8 + 2 * x], p[st * 8 + 2 * x + 1]);
                }
#pragma unroll
                for (int c = 0; c < HD / 32; ++c)
                    ak[c] = X::mma(frag_cols<S::NKC>(qt, u * 32 + st * 16, c * 32, lane), df, ak[c]);
                if constexpr (HDV > 0) {
                    if (a.gv || a.part_v) {
#pragma unroll
                        for (int c = 0; c < HDV / 32; ++c)
                            av[c] = X::mma(frag_cols<S::NVC>(gt, u * 32 + st * 16, c * 32, lane), pf, av[c]);
                    }
                }
            }
        }
        wait_fills();
        __syncthreads();
    }
    if (j >= nkeys) return;
    const float f = a.factor ? a.factor[0] : 1.f;
    auto put = [&](const fx16* acc, int n, float* part, const float* init, void* out, int C, float mul) {
#pragma unroll
        for (int c = 0; c < n; ++c)
#pragma unroll
            for (int x = 0; x < 16; x += 4) {
                const int ch = c * 32 + 2 * x + 4 * h;
                if (ch >= C) continue;
                float4 o = make_float4(acc[c][x], acc[c][x + 1], acc[c][x + 2], acc[c][x + 3]);
                if (!SINKS && init && j < a.init_keys && split == 0) {
                    const float4 z = *(const float4*)(init + (((int64_t)b * a.init_keys + j) * g.Hkv + hk) * C + ch);
                    o = make_float4(o.x + z.x, o.y + z.y, o.z + z.z, o.w + z.w);
                }
                if (part) {
                    *(float4*)(part + ((((int64_t)split * g.B + b) * nkeys + j) * g.Hkv + hk) * C + ch) = o;
                } else {
                    *(ix2*)((char*)out + ((((int64_t)b * g.Lk + j) * g.Hkv + hk) * C + ch) * 2) =
                        ix2{pack2<E>(o.x * mul, o.y * mul), pack2<E>(o.z * mul, o.w * mul)};
                }
            }
    };
    if (a.gk || a.part_k) put(ak, HD / 32, a.part_k, a.init_k, a.gk, g.C, g.scale * f / hot);
    if constexpr (HDV > 0) {
        if (a.gv || a.part_v) put(av, HDV / 32, a.part_v, a.init_v, a.gv, g.Cv, f);
    }
}

template <typename E, int HD, int HDV>
hipError_t go_q(const MatchGeo& g, const BwdArgs& a, hipStream_t s) {
    using S = BwdShape<HD, HDV>;
    const int row_tiles = (int)cdiv(g.rows(), 128);
    auto fn = k_match_bwd_q<E, HD, HDV>;
    hipError_t e = allow_lds((const void*)fn, S::kLdsQ);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(fn, dim3((unsigned)((int64_t)row_tiles * g.Hkv * g.B)), dim3(256), S::kLdsQ, s, g, a, row_tiles);
    return hipGetLastError();
}
template <typename E, int HD, int HDV, bool SINKS>
hipError_t go_k(const MatchGeo& g, const BwdArgs& a, int nsplit, hipStream_t s) {
    using S = BwdShape<HD, HDV>;
    const int key_tiles = (int)cdiv(SINKS && g.sinks < g.Lk ? g.sinks : g.Lk, 128);
    auto fn = k_match_bwd_k<E, HD, HDV, SINKS>;
    hipError_t e = allow_lds((const void*)fn, S::kLdsK);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(fn, dim3((unsigned)((int64_t)nsplit * key_tiles * g.Hkv * g.B)), dim3(256), S::kLdsK, s, g, a,
                       key_tiles, nsplit);
    return hipGetLastError();
}
template <int HD, int HDV>
hipError_t go_k_any(const MatchGeo& g, bool bf, const BwdArgs& a, bool sinks, int nsplit, hipStream_t s) {
    if constexpr (HDV > 0) {
        if (sinks) return bf ? go_k<__bf16, HD, HDV, true>(g, a, nsplit, s) : go_k<_Float16, HD, HDV, true>(g, a, nsplit, s);
    }
    return bf ? go_k<__bf16, HD, HDV, false>(g, a, nsplit, s) : go_k<_Float16, HD, HDV, false>(g, a, nsplit, s);
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
