// Forward of the row matching operators (match.h): one pass over the keys with the running maximum and sum
// of the softmax.  One workgroup = 4 waves; a wave owns 32 packed query rows (WK = 1) or, where there are few
// rows, the waves split each key tile between them and join at the end (WK > 1).  The next key tile is in
// flight into the other half of LDS while the present one is used.
//
//   attention      o = sum_j p_j v_j / sum_j p_j, lse = log sum_j exp(s_j)       (template HDV > 0)
//   cross entropy  lse and the target's score only                              (HDV = 0)
//
// P is rounded to the inputs' 16 bits for the product with V (each p off by at most half a step, their sum
// is kept in 32 bits); where the output is 32-bit it is split into two 16-bit parts, so that the product
// keeps the accuracy that the output can hold.
#include "match.h"
#include "match_launch.h"

namespace custma {
namespace {

template <int HD, int HDV, int WK>
struct FwdShape {
    static constexpr int WR = 4 / WK;                         // waves along rows
    static constexpr int BR = 32 * WR;                        // rows per workgroup
    static constexpr int KW = (WK == 1 && HD <= 128) ? 64 : 32;  // keys per wave and tile
    static constexpr int KT = KW * WK;
    static constexpr int NKC = HD / 8, NVC = HDV / 8;
    static constexpr int kTile = KT * (HD + HDV) * 2;         // bytes
    static constexpr int kJoin = WK > 1 ? 32 * WR * WK * 8 + (HDV ? 32 * WR * (WK - 1) * HDV * 4 : 4 * 32 * 4) : 0;
    static constexpr int kLds = 2 * kTile > kJoin ? 2 * kTile : kJoin;
};

template <typename E, int HD, int HDV, int WK, bool WIDE_OUT>
__global__ __launch_bounds__(256) void k_match_fwd(MatchGeo g, const char* __restrict__ q, const char* __restrict__ k,
                                                   const char* __restrict__ v, FwdOut o, int nsplit, int row_tiles) {
    using S = FwdShape<HD, HDV, WK>;
    typedef Half16<E> X;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = lane >> 5, col = lane & 31;
    const int wr = wave % S::WR, wk = wave / S::WR;

    // neighbouring workgroups share a key head's tiles: split fastest, then row tile, then head, then batch
    int64_t id = xcd_remap(blockIdx.x, gridDim.x);
    const int split = (int)(id % nsplit);
    id /= nsplit;
    const int rt = (int)(id % row_tiles);
    id /= row_tiles;
    const int hk = (int)(id % g.Hkv), b = (int)(id / g.Hkv);

    const int64_t off = g.offset ? g.offset[b] : 0;
    const int32_t len = key_length(g, b), rows = g.rows();
    const int r0 = rt * S::BR, r = r0 + wr * 32 + col;
    const int last = r0 + S::BR < rows ? r0 + S::BR - 1 : rows - 1;
    const Span first_s = span_of(g, off, len, r0 / g.G), last_s = span_of(g, off, len, last / g.G);
    const bool live = r < rows;
    const int i = (live ? r : rows - 1) / g.G, gh = (live ? r : rows - 1) % g.G;
    Span me = span_of(g, off, len, i);
    if (!live) me.lo = me.hi = 0;
    const int mysink = me.hi < g.sinks ? me.hi : g.sinks;
    // what the whole wave can see of the window: rows ascend, so do both bounds
    const int wlast = r0 + wr * 32 + 31 < rows ? r0 + wr * 32 + 31 : rows - 1;
    const bool wave_live = r0 + wr * 32 < rows;
    const Span wf = span_of(g, off, len, (wave_live ? r0 + wr * 32 : rows - 1) / g.G);
    const Span wl = span_of(g, off, len, wlast / g.G);
    const bool wave_full = r0 + wr * 32 + 31 < rows;

    // key tiles: sinks in front of the window, then the window
    int sink_end = g.sinks < first_s.lo ? g.sinks : first_s.lo;
    if (sink_end > last_s.hi) sink_end = last_s.hi;
    if (sink_end < 0) sink_end = 0;
    const int sink_tiles = (sink_end + S::KT - 1) / S::KT;
    const int win = last_s.hi > first_s.lo ? last_s.hi - first_s.lo : 0;
    const int tiles = sink_tiles + (win + S::KT - 1) / S::KT;
    const int t0 = (int)((int64_t)tiles * split / nsplit), t1 = (int)((int64_t)tiles * (split + 1) / nsplit);

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
    auto fill = [&](int t, int buf) {
        int ks, ke;
        tile_range(t, ks, ke);
        char* to = lds + buf * S::kTile;
        fill_tile<S::KT, S::NKC, 4>(to, kb, g.ks[1] * 2, ks, ke, kchunks, wave, lane);
        if constexpr (HDV > 0)
            fill_tile<S::KT, S::NVC, 4>(to + S::KT * HD * 2, vb, g.vs[1] * 2, ks, ke, vchunks, wave, lane);
    };
    if (t0 < t1) fill(t0, 0);

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
    const float sc = g.scale * kLog2e;
    int64_t target = -1;
    if constexpr (HDV == 0) {
        if (live) target = o.target[(int64_t)b * g.Lq + i];
        if (target < me.lo || target >= me.hi) target = -1;  // not a candidate: the row does not count
    }
    float m = -INFINITY, l = 0.f, picked = 0.f;
    fx16 acc[HDV ? HDV / 32 : 1];
#pragma unroll
    for (int c = 0; c < (HDV ? HDV / 32 : 1); ++c)
#pragma unroll
        for (int t = 0; t < 16; ++t) acc[c][t] = 0.f;

    wait_fills();
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1;
        if (t + 1 < t1) fill(t + 1, buf ^ 1);
        int ks, ke;
        tile_range(t, ks, ke);
        ks += wk * S::KW;  // this wave's keys of the tile
        const bool sink_tile = t < sink_tiles;
        if (wave_live && ks < ke && (sink_tile || (ks < wl.hi && (ks + S::KW > wf.lo || ks < g.sinks)))) {
            const char* kt = lds + buf * S::kTile;
            const char* vt = kt + S::KT * HD * 2;
            fx16 s[S::KW / 32];
#pragma unroll
            for (int u = 0; u < S::KW / 32; ++u) {
#pragma unroll
                for (int x = 0; x < 16; ++x) s[u][x] = 0.f;
#pragma unroll
                for (int st = 0; st < HD / 16; ++st)
                    s[u] = X::mma(frag_rows<S::NKC>(kt, wk * S::KW + u * 32, st, lane), qf[st], s[u]);
            }
            const bool all = !sink_tile && wave_full && ks >= wl.lo && ks + S::KW <= wf.hi;
            float mt = -INFINITY;
#pragma unroll
            for (int u = 0; u < S::KW / 32; ++u)
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    float z = s[u][x] * sc;
                    if (!all) {
                        const int j = ks + u * 32 + 8 * (x / 4) + 4 * h + x % 4;
                        const bool see = j < ke && j < me.hi && (j >= me.lo || j < mysink);
                        z = see ? z : -INFINITY;
                    }
                    s[u][x] = z;
                    mt = fmaxf(mt, z);
                }
            if constexpr (HDV == 0) {
                const int64_t tj = target - ks - 4 * h;  // target's place among this lane's scores
                if (__any(target >= ks && target < ks + S::KW)) {
#pragma unroll
                    for (int u = 0; u < S::KW / 32; ++u)
#pragma unroll
                        for (int x = 0; x < 16; ++x)
                            if (tj == u * 32 + 8 * (x / 4) + x % 4) picked = s[u][x];
                }
            }
            mt = fmaxf(mt, other_half(mt));
            const float mn = fmaxf(m, mt);
            const float base = mn == -INFINITY ? 0.f : mn;
            const float alpha = exp2_hw(m - base);
            m = mn;
            float sum = 0.f;
#pragma unroll
            for (int u = 0; u < S::KW / 32; ++u)
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const float p = exp2_hw(s[u][x] - base);
                    s[u][x] = p;
                    sum += p;
                }
            l = __builtin_fmaf(l, alpha, sum);
            if constexpr (HDV > 0) {
                if (__any(alpha != 1.f)) {
#pragma unroll
                    for (int c = 0; c < HDV / 32; ++c)
#pragma unroll
                        for (int x = 0; x < 16; ++x) acc[c][x] *= alpha;
                }
#pragma unroll
                for (int u = 0; u < S::KW / 32; ++u)
#pragma unroll
                    for (int st = 0; st < 2; ++st) {
                        ix4 pf, pl;
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const float a = s[u][st * 8 + 2 * x], c = s[u][st * 8 + 2 * x + 1];
                            pf[x] = pack2<E>(a, c);
                            if constexpr (WIDE_OUT) {
                                const fx2 back = unpack2<E>(pf[x]);
                                pl[x] = pack2<E>(a - back.x, c - back.y);
                            }
                        }
#pragma unroll
                        for (int c = 0; c < HDV / 32; ++c) {
                            const ix4 vf = frag_cols<S::NVC>(vt, wk * S::KW + u * 32 + st * 16, c * 32, lane);
                            acc[c] = X::mma(vf, pf, acc[c]);
                            if constexpr (WIDE_OUT) acc[c] = X::mma(vf, pl, acc[c]);
                        }
                    }
            }
        }
        wait_fills();
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
    if (!live) return;

    const int64_t row = ((int64_t)b * g.Lq + i) * g.heads() + hk * g.G + gh;
    if (nsplit > 1) {
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
        if (h == 0) {
            o.lse[row] = lse;
            o.loss[row] = target >= 0 ? (m - picked + __builtin_log2f(l)) * kLn2 : 0.f;
        }
    } else {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (h == 0 && o.lse) o.lse[row] = lse;
#pragma unroll
        for (int c = 0; c < HDV / 32; ++c)
#pragma unroll
            for (int x = 0; x < 16; x += 4) {
                const int ch = c * 32 + 2 * x + 4 * h;
                if (ch >= g.Cv) continue;
                const float a0 = acc[c][x] * inv, a1 = acc[c][x + 1] * inv, a2 = acc[c][x + 2] * inv,
                            a3 = acc[c][x + 3] * inv;
                if constexpr (WIDE_OUT) {
                    *(float4*)((float*)o.out + row * g.Cv + ch) = make_float4(a0, a1, a2, a3);
                } else {
                    const ix2 w = {pack2<E>(a0, a1), pack2<E>(a2, a3)};
                    *(ix2*)((char*)o.out + (row * g.Cv + ch) * 2) = w;
                    if (o.low) {
                        const fx2 u0 = unpack2<E>(w.x), u1 = unpack2<E>(w.y);
                        *(ix2*)((char*)o.low + (row * g.Cv + ch) * 2) =
                            ix2{pack2<E>(a0 - u0.x, a1 - u0.y), pack2<E>(a2 - u1.x, a3 - u1.y)};
                    }
                }
            }
    }
}

template <typename E, int HD, int HDV, int WK, bool WIDE_OUT>
hipError_t launch_shape(const MatchGeo& g, const void* q, const void* k, const void* v, const FwdOut& o, int nsplit,
                        hipStream_t s) {
    using S = FwdShape<HD, HDV, WK>;
    const int row_tiles = (int)cdiv(g.rows(), S::BR);
    const int64_t blocks = (int64_t)nsplit * row_tiles * g.Hkv * g.B;
    auto fn = k_match_fwd<E, HD, HDV, WK, WIDE_OUT>;
    hipError_t e = allow_lds((const void*)fn, S::kLds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(256), S::kLds, s, g, (const char*)q, (const char*)k,
                       (const char*)v, o, nsplit, row_tiles);
    return hipGetLastError();
}

template <int HD, int HDV>
hipError_t launch_hd(const MatchGeo& g, int dtype, bool wide_out, bool few, const void* q, const void* k,
                     const void* v, const FwdOut& o, int nsplit, hipStream_t s) {
    constexpr int WK = HD == 256 ? 2 : 4;
    const bool bf = dtype == CUSTMA_BF16;
#define CUSTMA_GO(E, W, O) return launch_shape<E, HD, HDV, W, O>(g, q, k, v, o, nsplit, s)
    if constexpr (HDV > 0) {
        if (wide_out) {
            if (few) { if (bf) CUSTMA_GO(__bf16, WK, true); else CUSTMA_GO(_Float16, WK, true); }
            else { if (bf) CUSTMA_GO(__bf16, 1, true); else CUSTMA_GO(_Float16, 1, true); }
        }
    }
    if (few) { if (bf) CUSTMA_GO(__bf16, WK, false); else CUSTMA_GO(_Float16, WK, false); }
    if (bf) CUSTMA_GO(__bf16, 1, false);
    CUSTMA_GO(_Float16, 1, false);
#undef CUSTMA_GO
}
}  // namespace

#define CUSTMA_CAT_(a, b) a##b
#define CUSTMA_CAT(a, b) CUSTMA_CAT_(a, b)
// one translation unit per channel count: -DCUSTMA_MATCH_HD=32/64/128/256
hipError_t CUSTMA_CAT(launch_match_fwd_, CUSTMA_MATCH_HD)(const MatchGeo& g, int dtype, bool wide_out, bool few, int hdv,
                                                         const void* q, const void* k, const void* v, const FwdOut& o,
                                                         int nsplit, hipStream_t s) {
    constexpr int HD = CUSTMA_MATCH_HD;
    if (hdv == 0) return launch_hd<HD, 0>(g, dtype, wide_out, few, q, k, v, o, nsplit, s);
    if (hdv == HD) return launch_hd<HD, HD>(g, dtype, wide_out, few, q, k, v, o, nsplit, s);
    if (HD > 32 && hdv == 32) return launch_hd<HD, 32>(g, dtype, wide_out, few, q, k, v, o, nsplit, s);
    return hipErrorInvalidValue;
}

}  // namespace custma
