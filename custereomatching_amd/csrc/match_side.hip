// The small passes around the row matching kernels (match.h): joining the parts of split key ranges and the
// sums of split row ranges, the output gradient in 16 bits, its product with the output, the loss's total.
// All are bound by memory or by launch; sums run in a fixed order.
#include "match.h"
#include "match_launch.h"

namespace custma {
namespace {
constexpr int kBlocks = 1024;

// one thread per 4 channels of a row (cross entropy: per row)
template <typename E, bool WIDE_OUT, bool LOSS>
__global__ __launch_bounds__(256) void k_join(MatchGeo g, FwdOut o, int nsplit, int64_t all) {
    const int per = LOSS ? 1 : g.Cv / 4;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= all * per) return;
    const int64_t row = id / per;
    const int ch = (int)(id % per) * 4;
    float M = -INFINITY;
    for (int s = 0; s < nsplit; ++s) M = fmaxf(M, o.part_ml[((int64_t)s * all + row) * 4]);
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f, picked = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < nsplit; ++s) {
        const float* ml = o.part_ml + ((int64_t)s * all + row) * 4;
        const float w = exp2_hw(ml[0] - base);
        L = __builtin_fmaf(w, ml[1], L);
        if constexpr (LOSS) {
            picked += ml[2];
        } else {
            const float4 v = *(const float4*)(o.part + ((int64_t)s * all + row) * g.Cv + ch);
            a[0] = __builtin_fmaf(w, v.x, a[0]);
            a[1] = __builtin_fmaf(w, v.y, a[1]);
            a[2] = __builtin_fmaf(w, v.z, a[2]);
            a[3] = __builtin_fmaf(w, v.w, a[3]);
        }
    }
    const float lse = L == 0.f ? -INFINITY : (M + __builtin_log2f(L)) * kLn2;
    if constexpr (LOSS) {
        const int b = (int)(row / g.Lq);
        const Span s = span_of(g, first_position(g, b), key_length(g, b), (int)(row % g.Lq));
        const int64_t t = o.target[row];
        o.lse[row] = lse;
        o.loss[row] = t >= s.lo && t < s.hi ? (M - picked + __builtin_log2f(L)) * kLn2 : 0.f;
    } else {
        if (ch == 0 && o.lse) o.lse[row] = lse;
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
        for (int x = 0; x < 4; ++x) a[x] *= inv;
        if constexpr (WIDE_OUT) {
            *(float4*)((float*)o.out + row * g.Cv + ch) = make_float4(a[0], a[1], a[2], a[3]);
        } else {
            const ix2 w = {pack2<E>(a[0], a[1]), pack2<E>(a[2], a[3])};
            *(ix2*)((char*)o.out + (row * g.Cv + ch) * 2) = w;
            if (o.low) {
                const fx2 u0 = unpack2<E>(w.x), u1 = unpack2<E>(w.y);
                *(ix2*)((char*)o.low + (row * g.Cv + ch) * 2) =
                    ix2{pack2<E>(a[0] - u0.x, a[1] - u0.y), pack2<E>(a[2] - u1.x, a[3] - u1.y)};
            }
        }
    }
}

template <typename T, typename Op>
__device__ __forceinline__ T block_reduce(T v, T* shared, Op op) {  // 256 threads; result in every thread
#pragma unroll
    for (int d = 32; d; d >>= 1) v = op(v, __shfl_xor(v, d, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    return op(op(shared[0], shared[1]), op(shared[2], shared[3]));
}

// the largest size of a finite value: one that is not finite must not move the others out of 16 bits
__device__ __forceinline__ float larger_finite(float m, float v) {
    v = fabsf(v);
    return v < INFINITY ? fmaxf(m, v) : m;
}
__global__ __launch_bounds__(256) void k_absmax(const float* __restrict__ x, int64_t n, float* __restrict__ part) {
    __shared__ float sh[4];
    float m = 0.f;
    const int64_t n4 = (uintptr_t)x % 16 == 0 ? n / 4 : 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += (int64_t)gridDim.x * 256) {
        const float4 v = ((const float4*)x)[i];
        m = larger_finite(larger_finite(larger_finite(larger_finite(m, v.x), v.y), v.z), v.w);
    }
    for (int64_t i = 4 * n4 + (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) m = larger_finite(m, x[i]);
    m = block_reduce(m, sh, [](float a, float b) { return fmaxf(a, b); });
    if (threadIdx.x == 0) part[blockIdx.x] = m;
}

// the power of two e with the largest of the parts in [2^(e-1), 2^e), at most 127; every thread of 256
__device__ __forceinline__ int exponent_of_parts(const float* part, int nparts, float* sh) {
    float m = 0.f;
    for (int i = threadIdx.x; i < nparts; i += 256) m = fmaxf(m, part[i]);
    m = block_reduce(m, sh, [](float a, float b) { return fmaxf(a, b); });
    int e = 0;
    if (m > 0.f) (void)frexpf(m, &e);
    return e < -120 ? -120 : e > 127 ? 127 : e;  // keeps 2^e normal and finite
}

// The rows' weights of a loss, the largest in [1, 2): the 16-bit product P * weight keeps its place, and the power of
// two comes back in 32 bits.
__global__ __launch_bounds__(256) void k_weights(const float* __restrict__ x, int64_t n, const float* __restrict__ part,
                                                 int nparts, const float* __restrict__ factor, float* __restrict__ out,
                                                 float* __restrict__ scale) {
    __shared__ float sh[4];
    const int e = x ? exponent_of_parts(part, nparts, sh) - 1 : 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) scale[0] = ldexpf(factor ? factor[0] : 1.f, e);
    const float f = ldexpf(1.f, -e);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[i] = x[i] * f;
}

// 32-bit output gradients in 16 bits, what the matrix units take: each off by half a step, and in float16 what is 2^-24
// of the largest is lost (one power of two for all: gradients of shared keys sum over rows, in one unit).
template <typename E>
__global__ __launch_bounds__(256) void k_narrow(const float* __restrict__ x, int64_t n4, const float* __restrict__ part,
                                                int nparts, ix2* __restrict__ out, float* __restrict__ scale) {
    __shared__ float sh[4];
    const int e = exponent_of_parts(part, nparts, sh);
    if (blockIdx.x == 0 && threadIdx.x == 0) scale[0] = ldexpf(1.f, e);
    const float f = ldexpf(1.f, -e);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += (int64_t)gridDim.x * 256) {
        const float4 v = ((const float4*)x)[i];
        out[i] = ix2{pack2<E>(v.x * f, v.y * f), pack2<E>(v.z * f, v.w * f)};
    }
}

// what the backward kernels keep per packed row; lpr lanes (a power of two >= Cv / 8) a row
template <typename E, bool OUT32, bool LOSS>
__global__ __launch_bounds__(256) void k_rows(MatchGeo g, BwdArgs a, int lpr_log, uint32_t all, const float* __restrict__ lse,
                                              const char* __restrict__ out, const char* __restrict__ low) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t at = id >> lpr_log;  // [B][Hkv][rows]
    const int lpr = 1 << lpr_log, c = (int)id & (lpr - 1), rows = g.rows(), Cv = g.Cv;
    const bool ok = at < all;
    const uint32_t at32 = ok ? (uint32_t)at : 0, bh = at32 / rows;
    const int r = (int)(at32 - bh * rows), hk = (int)(bh % g.Hkv), b = (int)(bh / g.Hkv);
    const int i = position_of_row(g, r);
    const int64_t row = ((int64_t)b * g.Lq + i) * g.heads() + hk * g.G + (r - i * g.G);
    float sum = 0.f;
    if constexpr (!LOSS) {
        if (ok && c < Cv / 8) {
            const ix4 gv = *(const ix4*)((const char*)a.go + (row * Cv + c * 8) * 2);
            float o[8];
            if constexpr (OUT32) {
                const float4 u = *(const float4*)(out + (row * Cv + c * 8) * 4);
                const float4 w = *(const float4*)(out + (row * Cv + c * 8) * 4 + 16);
                o[0] = u.x, o[1] = u.y, o[2] = u.z, o[3] = u.w, o[4] = w.x, o[5] = w.y, o[6] = w.z, o[7] = w.w;
            } else {
                const ix4 u4 = *(const ix4*)(out + (row * Cv + c * 8) * 2), w4 = *(const ix4*)(low + (row * Cv + c * 8) * 2);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const fx2 u = unpack2<E>(u4[x]), w = unpack2<E>(w4[x]);
                    o[2 * x] = u.x + w.x;
                    o[2 * x + 1] = u.y + w.y;
                }
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const fx2 u = unpack2<E>(gv[x]);
                sum = __builtin_fmaf(u.x, o[2 * x], sum);
                sum = __builtin_fmaf(u.y, o[2 * x + 1], sum);
            }
        }
        for (int d = lpr >> 1; d; d >>= 1) sum += __shfl_xor(sum, d, 64);
    }
    if (!ok || c != 0) return;
    float start = ((LOSS ? Half16<E>::kLift : 0.f) - lse[row] * kLog2e) / score_factor(g.scale);
    if constexpr (LOSS) {
        const Span s = span_of(g, first_position(g, b), key_length(g, b), i);
        const int64_t t = a.target[row];
        const bool counts = t >= s.lo && t < s.hi;
        const float weight = counts ? (a.weight ? a.weight[row] : 1.f) : 0.f;
        a.second[at] = weight;
        a.hot[at] = weight != 0.f ? (int)t : -1;
        if (weight == 0.f) start = -INFINITY;
    } else {
        a.second[at] = -sum;
    }
    a.start[at] = start;
}

struct SumArgs {
    const float* part;
    int64_t n4;      // groups of four values of one split
    char* out;
    float scale;
};
// sums over row splits, of two tensors (the second may have n4 = 0)
template <typename E>
__global__ __launch_bounds__(256) void k_sum(SumArgs x, SumArgs y, int nsplit, bool to32, const float* __restrict__ factor) {
    const float f = factor ? factor[0] : 1.f;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < x.n4 + y.n4; i += (int64_t)gridDim.x * 256) {
        const bool second = i >= x.n4;
        const SumArgs& z = second ? y : x;
        const int64_t e = second ? i - x.n4 : i;
        const float4* p = (const float4*)z.part + e;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        int s = 0;
        for (; s + 8 <= nsplit; s += 8) {  // eight in flight, added in order
            float4 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = p[(int64_t)(s + u) * z.n4];
#pragma unroll
            for (int u = 0; u < 8; ++u) a = make_float4(a.x + v[u].x, a.y + v[u].y, a.z + v[u].z, a.w + v[u].w);
        }
        for (; s < nsplit; ++s) {
            const float4 v = p[(int64_t)s * z.n4];
            a = make_float4(a.x + v.x, a.y + v.y, a.z + v.z, a.w + v.w);
        }
        const float m = f * z.scale;
        if (to32) ((float4*)z.out)[e] = a;
        else ((ix2*)z.out)[e] = ix2{pack2<E>(a.x * m, a.y * m), pack2<E>(a.z * m, a.w * m)};
    }
}

__global__ __launch_bounds__(256) void k_total_parts(const float* __restrict__ loss, const int64_t* __restrict__ target,
                                                     MatchGeo g, int64_t n, double* __restrict__ part) {
    __shared__ double sh[4];
    double sum = 0., count = 0.;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const uint32_t b = (uint32_t)i / (uint32_t)g.Lq;  // rows of a call are below 2^32
        const Span s = span_of(g, 0, g.Lk, (int)((uint32_t)i - b * (uint32_t)g.Lq));
        const int64_t t = target[i];
        if (t >= s.lo && t < s.hi) {
            sum += loss[i];
            count += 1.;
        }
    }
    sum = block_reduce(sum, sh, [](double a, double b) { return a + b; });
    count = block_reduce(count, sh, [](double a, double b) { return a + b; });
    if (threadIdx.x == 0) {
        part[2 * blockIdx.x] = sum;
        part[2 * blockIdx.x + 1] = count;
    }
}
__global__ __launch_bounds__(256) void k_total(const double* __restrict__ part, int nparts, float* __restrict__ total) {
    __shared__ double sh[4];
    double sum = 0., count = 0.;
    for (int i = threadIdx.x; i < nparts; i += 256) {
        sum += part[2 * i];
        count += part[2 * i + 1];
    }
    sum = block_reduce(sum, sh, [](double a, double b) { return a + b; });
    count = block_reduce(count, sh, [](double a, double b) { return a + b; });
    if (threadIdx.x == 0) {
        const double inv = 1. / (count > 1. ? count : 1.);
        total[0] = (float)sum;
        total[1] = (float)inv;
        total[2] = (float)(sum * inv);
    }
}

int blocks_for(int64_t threads) {
    const int64_t b = cdiv(threads, 256);
    return (int)(b < kBlocks ? (b < 1 ? 1 : b) : kBlocks);
}
}  // namespace

hipError_t launch_match_join(const MatchGeo& g, int dtype, bool wide_out, const FwdOut& o, int nsplit, hipStream_t s) {
    const int64_t all = (int64_t)g.B * g.Lq * g.heads();
    const bool loss = o.loss != nullptr, bf = dtype == CUSTMA_BF16;
    const dim3 grid((unsigned)cdiv(all * (loss ? 1 : g.Cv / 4), 256));
    if (loss) hipLaunchKernelGGL((k_join<__bf16, true, true>), grid, dim3(256), 0, s, g, o, nsplit, all);
    else if (wide_out) hipLaunchKernelGGL((k_join<__bf16, true, false>), grid, dim3(256), 0, s, g, o, nsplit, all);
    else if (bf) hipLaunchKernelGGL((k_join<__bf16, false, false>), grid, dim3(256), 0, s, g, o, nsplit, all);
    else hipLaunchKernelGGL((k_join<_Float16, false, false>), grid, dim3(256), 0, s, g, o, nsplit, all);
    return hipGetLastError();
}

hipError_t launch_match_narrow(const float* go, int64_t n, int dtype, void* out16, float* scale, float* partials,
                               hipStream_t s) {
    const int blocks = blocks_for(n / 4);
    hipLaunchKernelGGL(k_absmax, dim3(blocks), dim3(256), 0, s, go, n, partials);
    if (dtype == CUSTMA_BF16)
        hipLaunchKernelGGL(k_narrow<__bf16>, dim3(blocks), dim3(256), 0, s, go, n / 4, partials, blocks, (ix2*)out16, scale);
    else
        hipLaunchKernelGGL(k_narrow<_Float16>, dim3(blocks), dim3(256), 0, s, go, n / 4, partials, blocks, (ix2*)out16, scale);
    return hipGetLastError();
}

hipError_t launch_match_weights(const float* weight, int64_t n, const float* factor, float* out, float* scale,
                                float* partials, hipStream_t s) {
    const int blocks = weight ? blocks_for(n) : 1;
    if (weight) hipLaunchKernelGGL(k_absmax, dim3(blocks), dim3(256), 0, s, weight, n, partials);
    hipLaunchKernelGGL(k_weights, dim3(blocks), dim3(256), 0, s, weight, weight ? n : 0, partials, blocks, factor, out, scale);
    return hipGetLastError();
}

hipError_t launch_match_rows(const MatchGeo& g, int dtype, const BwdArgs& a, const float* lse, const void* out,
                             bool out_f32, const void* low, hipStream_t s) {
    const int64_t all = (int64_t)g.B * g.Lq * g.heads();
    int log = 0;
    while (out && (1 << log) < g.Cv / 8) ++log;
    const dim3 grid((unsigned)cdiv(all << log, 256));
    const bool bf = dtype == CUSTMA_BF16;
#define CUSTMA_GO(E, O, L) \
    hipLaunchKernelGGL((k_rows<E, O, L>), grid, dim3(256), 0, s, g, a, log, (uint32_t)all, lse, (const char*)out, (const char*)low)
    if (!out) { if (bf) CUSTMA_GO(__bf16, false, true); else CUSTMA_GO(_Float16, false, true); }
    else if (out_f32) { if (bf) CUSTMA_GO(__bf16, true, false); else CUSTMA_GO(_Float16, true, false); }
    else { if (bf) CUSTMA_GO(__bf16, false, false); else CUSTMA_GO(_Float16, false, false); }
#undef CUSTMA_GO
    return hipGetLastError();
}

hipError_t launch_match_sum(const float* part, int nsplit, int64_t n, int dtype, bool to32, const float* factor,
                            float scale, void* out, const float* part2, int64_t n2, float scale2, void* out2, hipStream_t s) {
    if (!out) n = 0;
    if (!out2) n2 = 0;
    if (n + n2 == 0) return hipSuccess;
    const int64_t b = cdiv((n + n2) / 4, 256);
    const dim3 grid((unsigned)(b < 8192 ? b : 8192));
    const SumArgs x{part, n / 4, (char*)out, scale}, y{part2, n2 / 4, (char*)out2, scale2};
    if (dtype == CUSTMA_BF16) hipLaunchKernelGGL(k_sum<__bf16>, grid, dim3(256), 0, s, x, y, nsplit, to32, factor);
    else hipLaunchKernelGGL(k_sum<_Float16>, grid, dim3(256), 0, s, x, y, nsplit, to32, factor);
    return hipGetLastError();
}

hipError_t launch_match_total(const float* loss, const int64_t* target, const MatchGeo& g, int64_t n, float* total,
                              double* partials, hipStream_t s) {
    const int blocks = blocks_for(n);
    hipLaunchKernelGGL(k_total_parts, dim3(blocks), dim3(256), 0, s, loss, target, g, n, partials);
    hipLaunchKernelGGL(k_total, dim3(1), dim3(256), 0, s, partials, blocks, total);
    return hipGetLastError();
}

}  // namespace custma
