// Cross entropy over classes with wide vectors (more channels than match_fwd.hip holds in registers), every
// class visible.  The scores are a matrix product that is never stored:
//   forward   k_wide_scores walks a range of the classes in 256 x 256 tiles of the product and keeps each
//             query's running maximum and sum; the ranges are joined afterwards.
//   backward  the classes are taken in pieces.  Per piece k_wide_scores computes the product again and writes
//             dz = w (P - [target]) of the piece in 16 bits, then two products use it:
//             dx += dz W (32-bit sums over the pieces), dW = dz^T x.
//             16 bits are what the matrix units take; its rounding stays below that of the gradients (bfloat16: both are
//             off by 1.66e-3 of their norm, as the formula in 32 bits rounded once is).
// 8 waves a workgroup, each 128 x 64 of the tile (4 x 2 matrix instructions of 32 x 32 a step): 6 KiB of
// operands from LDS feed 8 instructions, so that LDS is read at three quarters of its rate.  64 channels a
// step, the next step's tiles in flight.
//
// Bound by the matrix instructions, which run 49 % of the time (scores), 43 % (dx) and 48 % (dW): 4093 rows, 50021
// classes, 1024 channels take 0.48 ms for the loss (870 TFLOP/s) and 1.6 ms for both gradients (800 TFLOP/s over
// their three products); a large library product reaches 1400.  333 rows, 128000 classes, 512 channels, loss only:
// 82 us and 5 for the join, where reading the classes once takes 28.  The backward's scores spill 44 bytes a lane.
#include <type_traits>

#include "match.h"
#include "match_launch.h"

namespace custma {
namespace {
constexpr int kTM = 256, kTN = 256, kTK = 64, kWaves = 8;
constexpr int kStage = (kTM + kTN) * kTK * 2;
constexpr int64_t kPieceBytes = (int64_t)128 << 20;  // dz of one piece
constexpr int64_t kJoinBlocks = 1 << 20;             // a launch counts its threads in 32 bits
constexpr int kTargetBlocks = 256;                   // one workgroup a compute unit (128 KiB of LDS)

template <typename E>
struct Tile {  // a wave's part of the product
    fx16 acc[4][2];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int x = 0; x < 16; ++x) acc[m][n][x] = 0.f;
    }
    template <typename FA, typename FB>
    __device__ __forceinline__ void step(FA fa, FB fb) {
#pragma unroll
        for (int st = 0; st < kTK / 16; ++st) {
            ix4 a[4], b[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) b[n] = fb(st, n);
#pragma unroll
            for (int m = 0; m < 4; ++m) a[m] = fa(st, m);
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int n = 0; n < 2; ++n) acc[m][n] = Half16<E>::mma(a[m], b[n], acc[m][n]);
        }
    }
};

struct WideArgs {
    const char *q, *k;       // rows of one batch entry
    int64_t qs, ks;          // bytes between rows
    const int64_t* target;
    const float *lse, *weight;
    float* part;             // forward: [2 nsplit][all rows][4]
    char* dz;                // backward: [N][pitch]
    int64_t row0, all;       // first row of the entry, rows of all entries
    int32_t N, V, C;
    int32_t v0, pitch;       // backward: first class and padded width of the piece
    float sc;
};

template <typename E, bool BWD>
__global__ __launch_bounds__(512) void k_wide_scores(WideArgs w, int row_tiles, int nsplit) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = lane >> 5, col = lane & 31, wm = wave & 1, wn = wave >> 1;
    uint32_t id = xcd_block();
    const int rt = (int)split_off(id, row_tiles), split = (int)id;
    const int n0 = rt * kTN;
    const int v_end = BWD ? (w.v0 + w.pitch < w.V ? w.v0 + w.pitch : w.V) : w.V;
    const int tiles_all = BWD ? w.pitch / kTM : (w.V + kTM - 1) / kTM;
    const int t0 = (int)((uint64_t)tiles_all * split / nsplit), t1 = (int)((uint64_t)tiles_all * (split + 1) / nsplit);
    const int ksteps = (w.C + kTK - 1) / kTK, chunks = w.C / 8;
    const int first = BWD ? w.v0 : 0;

    auto fill = [&](int t, int ks, int buf) {
        const uint32_t to = lds_offset(lds) + buf * kStage;
        const int left = chunks - ks * (kTK / 8);
        fill_tile<kTM, kTK / 8, kWaves>(to, w.k + ks * kTK * 2, w.ks, first + t * kTM, v_end, left, wave, lane);
        fill_tile<kTN, kTK / 8, kWaves>(to + kTM * kTK * 2, w.q + ks * kTK * 2, w.qs, n0, w.N, left, wave, lane);
    };
    int n[2];
    bool live[2];
    int target[2];
    float m[2], l[2], picked[2], base[2], weight[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        n[c] = n0 + wn * 64 + c * 32 + col;
        live[c] = n[c] < w.N;
        const int64_t t = live[c] ? w.target[w.row0 + n[c]] : -1;
        target[c] = t >= 0 && t < w.V ? (int)t : -1;
        m[c] = -INFINITY;
        l[c] = picked[c] = base[c] = weight[c] = 0.f;
        if constexpr (BWD) {
            if (live[c]) {
                base[c] = w.lse[w.row0 + n[c]] * kLog2e - Half16<E>::kLift;
                weight[c] = target[c] < 0 ? 0.f : w.weight ? w.weight[w.row0 + n[c]] : 1.f;
            }
        }
    }
    const float hot = __builtin_ldexpf(1.f, (int)Half16<E>::kLift);
    Tile<E> d;
    if (t0 < t1) fill(t0, 0, 0);
    wait_fills();
    __syncthreads();
    int buf = 0;
    for (int t = t0; t < t1; ++t) {
        d.zero();
        for (int ks = 0; ks < ksteps; ++ks, buf ^= 1) {
            if (ks + 1 < ksteps) fill(t, ks + 1, buf ^ 1);
            else if (t + 1 < t1) fill(t + 1, 0, buf ^ 1);
            const char* at = lds + buf * kStage;
            const char* bt = at + kTM * kTK * 2;
            d.step([&](int st, int x) { return frag_rows<kTK / 8>(at, wm * 128 + x * 32, st, lane); },
                   [&](int st, int x) { return frag_rows<kTK / 8>(bt, wn * 64 + x * 32, st, lane); });
            wait_fills();
            __syncthreads();
        }
        const int vw = first + t * kTM + wm * 128;  // the wave's first class
        if constexpr (BWD) {
            // through the LDS buffer that the next tile's first step is not in, 32 queries at a time
            char* mine = lds + (buf ^ 1) * kStage + wave * 32 * 128 * 2;
            const bool whole = vw + 128 <= w.V;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int tj = target[c] - vw - 4 * h;
                const bool hit = __any(target[c] >= vw && target[c] < vw + 128);
                fx16 o[4];
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const int at = r * 32 + 8 * (x / 4) + x % 4;
                        float p = exp2_hw(__builtin_fmaf(d.acc[r][c][x], w.sc, -base[c]));
                        if (hit && tj == at) p -= hot;
                        p *= weight[c];
                        if (!whole && vw + 4 * h + at >= w.V) p = 0.f;
                        o[r][x] = weight[c] == 0.f ? 0.f : p;
                    }
                __builtin_amdgcn_wave_barrier();
                store_rows<E, 16>(mine, o, 1.f, 128, lane, [&](int x) -> char* {
                    const int q = n0 + wn * 64 + c * 32 + x;
                    return q < w.N ? w.dz + ((int64_t)q * w.pitch + (vw - first)) * 2 : nullptr;
                });
            }
            __syncthreads();  // that buffer is filled again next
        } else {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int tj = target[c] - vw - 4 * h;
                const bool whole = vw + 128 <= w.V;
                const bool hit = __any(target[c] >= vw && target[c] < vw + 128);
                float mt = -INFINITY;
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const int at = r * 32 + 8 * (x / 4) + x % 4;
                        float z = d.acc[r][c][x] * w.sc;
                        if (!whole && vw + 4 * h + at >= w.V) z = -INFINITY;
                        if (hit && tj == at) picked[c] = z;
                        d.acc[r][c][x] = z;
                        mt = fmaxf(mt, z);
                    }
                mt = fmaxf(mt, other_half(mt));
                const float mn = fmaxf(m[c], mt), b0 = mn == -INFINITY ? 0.f : mn;
                float sum = 0.f;
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int x = 0; x < 16; ++x) sum += exp2_hw(d.acc[r][c][x] - b0);
                l[c] = __builtin_fmaf(l[c], exp2_hw(m[c] - b0), sum);
                m[c] = mn;
            }
        }
    }
    if constexpr (!BWD) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const float lt = l[c] + other_half(l[c]), pt = picked[c] + other_half(picked[c]);
            if (live[c] && h == 0)
                *(float4*)(w.part + (((int64_t)split * 2 + wm) * w.all + w.row0 + n[c]) * 4) = make_float4(m[c], lt, pt, 0.f);
        }
    }
}

// D[n][m] = sum_k A[k][m] B(k, n): A rows are the contraction; B's rows are n (dx) or the contraction (dW).
//
// Queries that do not count have rows of zeros in dz, but 0 * inf is not 0.  dx writes zeros for them (a class may hold
// an inf).  dW looks at its sums at the end, and where one is not finite it runs again with those queries' vectors as
// zeros: what is not finite then belongs to queries that count.
struct GemmArgs {
    const char *a, *b;
    int64_t as, bs;      // bytes between rows
    int32_t M, N, K;
    float* d32;          // [splits][N][M], added to where `add`
    char* d16;           // or 16-bit [N][M]
    const float* factor;
    float scale;
    int32_t add;
    const int64_t* target;  // of the queries
    const float* weight;    // of the queries; null: 1
    int32_t classes;
    __device__ __forceinline__ bool counts(int q) const {
        const int64_t t = target[q];
        return t >= 0 && t < classes && (!weight || weight[q] != 0.f);
    }
};

template <typename E, bool B_ROWS>
__global__ __launch_bounds__(512) void k_wide_gemm(GemmArgs w, int m_tiles, int n_tiles, int nsplit) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = lane >> 5, col = lane & 31, wm = wave & 1, wn = wave >> 1;
    uint32_t id = xcd_block();
    const int mt = (int)split_off(id, m_tiles), nt = (int)split_off(id, n_tiles), split = (int)id;
    const int m0 = mt * kTM, n0 = nt * kTN;
    const int steps = (w.K + kTK - 1) / kTK;
    const int s0 = (int)((int64_t)steps * split / nsplit), s1 = (int)((int64_t)steps * (split + 1) / nsplit);
    Tile<E> d;
    auto walk = [&](auto careful_c) __attribute__((always_inline)) {
        constexpr bool CAREFUL = decltype(careful_c)::value;
        auto fill = [&](int ks, int buf) __attribute__((always_inline)) {
            const uint32_t to = lds_offset(lds) + buf * kStage;
            if constexpr (CAREFUL)
                fill_rows<kTK, kTM / 8, kWaves>(
                    to,
                    [&](int t) -> const char* {
                        const int q = ks * kTK + t;
                        return q < w.K && w.counts(q) ? w.a + m0 * 2 + (int64_t)q * w.as : nullptr;
                    },
                    w.M / 8 - m0 / 8, wave, lane);
            else
                fill_tile<kTK, kTM / 8, kWaves>(to, w.a + m0 * 2, w.as, ks * kTK, w.K, w.M / 8 - m0 / 8, wave, lane);
            if constexpr (B_ROWS)
                fill_tile<kTN, kTK / 8, kWaves>(to + kTM * kTK * 2, w.b + (int64_t)ks * kTK * 2, w.bs, n0, w.N, kTK / 8, wave, lane);
            else
                fill_tile<kTK, kTN / 8, kWaves>(to + kTM * kTK * 2, w.b + (int64_t)n0 * 2, w.bs, ks * kTK, w.K, kTN / 8, wave, lane);
        };
        d.zero();
        if (s0 < s1) fill(s0, 0);
        wait_fills();
        __syncthreads();
        for (int ks = s0; ks < s1; ++ks) {
            const int buf = (ks - s0) & 1;
            if (ks + 1 < s1) fill(ks + 1, buf ^ 1);
            const char* at = lds + buf * kStage;
            const char* bt = at + kTM * kTK * 2;
            if constexpr (B_ROWS)
                d.step([&](int st, int x) { return frag_cols_plain<kTM / 8>(at, st * 16, wm * 128 + x * 32, lane); },
                       [&](int st, int x) { return frag_rows<kTK / 8>(bt, wn * 64 + x * 32, st, lane); });
            else
                d.step([&](int st, int x) { return frag_cols<kTM / 8>(at, st * 16, wm * 128 + x * 32, lane); },
                       [&](int st, int x) { return frag_cols<kTN / 8>(bt, st * 16, wn * 64 + x * 32, lane); });
            wait_fills();
            __syncthreads();
        }
    };
    walk(std::false_type{});
    if constexpr (!B_ROWS) {
        bool bad = false;
#pragma unroll
        for (int r = 0; r < 4; ++r) bad |= any_not_finite(d.acc[r], 0.f);
        if (__syncthreads_or(bad)) walk(std::true_type{});
    }
    const float f = w.scale * (w.factor ? w.factor[0] : 1.f);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int n = n0 + wn * 64 + c * 32 + col;
        if (n >= w.N) continue;
        const bool drop = B_ROWS && !w.counts(n);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int x = 0; x < 16; x += 4) {
                const int m = m0 + wm * 128 + r * 32 + 2 * x + 4 * h;
                if (m >= w.M) continue;
                float4 o = make_float4(d.acc[r][c][x], d.acc[r][c][x + 1], d.acc[r][c][x + 2], d.acc[r][c][x + 3]);
                if (drop) o = make_float4(0.f, 0.f, 0.f, 0.f);
                if (w.d32) {
                    float4* to = (float4*)(w.d32 + ((int64_t)split * w.N + n) * w.M + m);
                    if (w.add) {
                        const float4 z = *to;
                        o = make_float4(o.x + z.x, o.y + z.y, o.z + z.z, o.w + z.w);
                    }
                    *to = o;
                } else {
                    *(ix2*)(w.d16 + ((int64_t)n * w.M + m) * 2) = ix2{pack2<E>(o.x * f, o.y * f), pack2<E>(o.z * f, o.w * f)};
                }
            }
    }
}

// joins the forward's parts: 4 rows at a time, 64 threads each
__global__ __launch_bounds__(256) void k_wide_join(MatchGeo g, FwdOut o, int nparts, int64_t all) {
    __shared__ float sh[3][4][64];
    const int x = threadIdx.x & 3, p = threadIdx.x >> 2;
    for (int64_t row0 = (int64_t)blockIdx.x * 4; row0 < all; row0 += (int64_t)gridDim.x * 4) {
        const int64_t row = row0 + x;
        float m = -INFINITY, l = 0.f, picked = 0.f;
        if (row < all) {
            for (int s = p; s < nparts; s += 64) {
                const float4 v = *(const float4*)(o.part_ml + ((int64_t)s * all + row) * 4);
                const float mn = fmaxf(m, v.x), b = mn == -INFINITY ? 0.f : mn;
                l = l * exp2_hw(m - b) + v.y * exp2_hw(v.x - b);
                m = mn;
                picked += v.z;
            }
        }
        __syncthreads();  // the rows before have been read
        sh[0][x][p] = m, sh[1][x][p] = l, sh[2][x][p] = picked;
        __syncthreads();
        if (threadIdx.x >= 4 || row >= all) continue;
        float M = -INFINITY;
        for (int s = 0; s < 64; ++s) M = fmaxf(M, sh[0][x][s]);
        const float b = M == -INFINITY ? 0.f : M;
        float L = 0.f, P = 0.f;
        for (int s = 0; s < 64; ++s) {
            L = __builtin_fmaf(sh[1][x][s], exp2_hw(sh[0][x][s] - b), L);
            P += sh[2][x][s];
        }
        const int64_t t = o.target[row];
        o.lse[row] = L == 0.f ? -INFINITY : (M + __builtin_log2f(L)) * kLn2;
        o.loss[row] = t >= 0 && t < g.Lk ? (M - P + __builtin_log2f(L)) * kLn2 : 0.f;
    }
}

int wide_pitch(const MatchGeo& g) {
    const int64_t whole = cdiv(g.Lk, kTM) * kTM;
    int64_t p = kPieceBytes / 2 / (g.Lq > 0 ? g.Lq : 1) / kTM * kTM;
    if (p < 4 * kTM) p = 4 * kTM;
    return (int)(p < whole ? p : whole);
}
int dx_splits(const MatchGeo& g) {
    const int64_t blocks = cdiv(g.Lq, kTN) * cdiv(g.C, kTM);
    int64_t s = blocks ? kTargetBlocks / blocks : 1;
    const int64_t most = wide_pitch(g) / kTK / 4;  // at least four steps each
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

template <typename E>
hipError_t bwd_entry(const MatchGeo& g, const BwdArgs& a, int b, char* dz, float* part, hipStream_t s) {
    const int pitch = wide_pitch(g), S = dx_splits(g);
    const int row_tiles = (int)cdiv(g.Lq, kTN), c_tiles = (int)cdiv(g.C, kTM);
    const int esz = 2;
    hipError_t e;
    static std::atomic<uint64_t> done[3];
    if ((e = allow_lds((const void*)k_wide_scores<E, true>, 2 * kStage, done[0])) != hipSuccess) return e;
    if ((e = allow_lds((const void*)k_wide_gemm<E, true>, 2 * kStage, done[1])) != hipSuccess) return e;
    if ((e = allow_lds((const void*)k_wide_gemm<E, false>, 2 * kStage, done[2])) != hipSuccess) return e;
    WideArgs w{};
    w.q = (const char*)a.q + (int64_t)b * g.qs[0] * esz;
    w.k = (const char*)a.k + (int64_t)b * g.ks[0] * esz;
    w.qs = g.qs[1] * esz, w.ks = g.ks[1] * esz;
    w.target = a.target, w.lse = a.lse, w.weight = a.weight;
    w.dz = dz, w.pitch = pitch;
    w.row0 = (int64_t)b * g.Lq, w.all = (int64_t)g.B * g.Lq;
    w.N = g.Lq, w.V = g.Lk, w.C = g.C;
    w.sc = g.scale * kLog2e;
    const float out_scale = g.scale / ldexpf(1.f, (int)Half16<E>::kLift);
    for (int v0 = 0; v0 < g.Lk; v0 += pitch) {
        w.v0 = v0;
        const int ctiles = pitch / kTM, want = (int)cdiv(kTargetBlocks, row_tiles), splits = want < ctiles ? want : ctiles;
        hipLaunchKernelGGL((k_wide_scores<E, true>), dim3(row_tiles * splits), dim3(512), 2 * kStage, s, w, row_tiles, splits);
        const int V = g.Lk - v0 < pitch ? g.Lk - v0 : pitch;
        if (a.gq) {
            GemmArgs x{};
            x.a = w.k + (int64_t)v0 * w.ks, x.as = w.ks, x.b = dz, x.bs = (int64_t)pitch * 2;
            x.M = g.C, x.N = g.Lq, x.K = V;
            x.d32 = part, x.add = v0 > 0;
            x.target = a.target + w.row0, x.weight = a.weight ? a.weight + w.row0 : nullptr, x.classes = g.Lk;
            hipLaunchKernelGGL((k_wide_gemm<E, true>), dim3(c_tiles * row_tiles * S), dim3(512), 2 * kStage, s, x, c_tiles, row_tiles, S);
        }
        if (a.gk) {
            GemmArgs x{};
            x.a = w.q, x.as = w.qs, x.b = dz, x.bs = (int64_t)pitch * 2;
            x.M = g.C, x.N = V, x.K = g.Lq;
            x.d16 = (char*)a.gk + ((int64_t)b * g.Lk + v0) * g.C * 2;
            x.factor = a.factor, x.scale = out_scale;
            x.target = a.target + w.row0, x.weight = a.weight ? a.weight + w.row0 : nullptr, x.classes = g.Lk;
            const int n_tiles = (int)cdiv(V, kTN);
            hipLaunchKernelGGL((k_wide_gemm<E, false>), dim3(c_tiles * n_tiles), dim3(512), 2 * kStage, s, x, c_tiles, n_tiles, 1);
        }
    }
    if (a.gq)
        e = launch_match_sum(part, S, (int64_t)g.Lq * g.C, sizeof(E) == 2 && Half16<E>::kLift == 0.f ? CUSTMA_BF16 : CUSTMA_F16,
                             false, a.factor, out_scale, (char*)a.gq + (int64_t)b * g.Lq * g.C * 2, nullptr, 0, 1.f, nullptr, s);
    return e != hipSuccess ? e : hipGetLastError();
}
}  // namespace

int wide_splits(const MatchGeo& g) {
    const int64_t tiles = cdiv(g.Lk, kTM), row_tiles = cdiv(g.Lq, kTN);
    int64_t s = row_tiles ? cdiv(kTargetBlocks, row_tiles) : 1;
    if (s > tiles) s = tiles;
    return (int)(s < 1 ? 1 : s);  // without classes too: the rows' results are written all the same
}

hipError_t launch_wide_fwd(const MatchGeo& g, int dtype, const void* q, const void* k, const FwdOut& o, hipStream_t s) {
    const int nsplit = wide_splits(g), row_tiles = (int)cdiv(g.Lq, kTN);
    const bool bf = dtype == CUSTMA_BF16;
    const void* fn = bf ? (const void*)k_wide_scores<__bf16, false> : (const void*)k_wide_scores<_Float16, false>;
    static std::atomic<uint64_t> done[2];
    hipError_t e = allow_lds(fn, 2 * kStage, done[bf]);
    if (e != hipSuccess) return e;
    for (int b = 0; b < g.B; ++b) {
        WideArgs w{};
        w.q = (const char*)q + (int64_t)b * g.qs[0] * 2;
        w.k = (const char*)k + (int64_t)b * g.ks[0] * 2;
        w.qs = g.qs[1] * 2, w.ks = g.ks[1] * 2;
        w.target = o.target;
        w.part = o.part_ml;
        w.row0 = (int64_t)b * g.Lq, w.all = (int64_t)g.B * g.Lq;
        w.N = g.Lq, w.V = g.Lk, w.C = g.C;
        w.sc = g.scale * kLog2e;
        if (bf) hipLaunchKernelGGL((k_wide_scores<__bf16, false>), dim3(row_tiles * nsplit), dim3(512), 2 * kStage, s, w, row_tiles, nsplit);
        else hipLaunchKernelGGL((k_wide_scores<_Float16, false>), dim3(row_tiles * nsplit), dim3(512), 2 * kStage, s, w, row_tiles, nsplit);
    }
    const int64_t all = (int64_t)g.B * g.Lq;
    const int64_t blocks = cdiv(all, 4);
    hipLaunchKernelGGL(k_wide_join, dim3((unsigned)(blocks < kJoinBlocks ? blocks : kJoinBlocks)), dim3(256), 0, s, g, o, 2 * nsplit, all);
    return hipGetLastError();
}

size_t wide_bwd_bytes(const MatchGeo& g) {
    return up256((size_t)g.Lq * wide_pitch(g) * 2) + up256((size_t)dx_splits(g) * g.Lq * g.C * 4);
}

hipError_t launch_wide_bwd(const MatchGeo& g, int dtype, const BwdArgs& a, void* ws, hipStream_t s) {
    char* dz = (char*)ws;
    float* part = (float*)(dz + up256((size_t)g.Lq * wide_pitch(g) * 2));
    for (int b = 0; b < g.B; ++b) {
        const hipError_t e = dtype == CUSTMA_BF16 ? bwd_entry<__bf16>(g, a, b, dz, part, s) : bwd_entry<_Float16>(g, a, b, dz, part, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace custma
