// Patch descriptors: the centred, unit-norm k x k patch of every pixel as a vector of k * k channels, so that
// the dot product of a camera and a projector descriptor is their ZNCC.  Patches as in the cost volume
// (zero-padded, taps at offsets -k/2 .. k-1-k/2), epsilon under the root as there (per vector: ss + 1e-8).
//   x_t = I[p + o_t],  m = mean x,  s = 1 / sqrt(sum (x - m)^2 + eps),  d_t = s (x_t - m)
// Channels are padded with zeros to a multiple of 8 (16 bytes).  Taps are taken relative to the patch's
// centre before they are summed: a flat patch gives exact zeros.
//
// Backward.  With a = sum_t g_t d_t and b = mean g,  dI[p] = sum over pixels q whose patch holds p, t = p - q, of
//   s g_t - s b - s^2 a (I[p] - m).
// The last two need only sums over q of s^2 a and of s^2 a m - s b (kept in 64 bits: around flat patches s
// is 1e4 and they cancel), so every g is read from memory once.  A workgroup walks down a strip of 64 columns;
// each thread owns a column and every fourth of the k image rows that are open at a time, in registers: one
// owner per sum, no atomics.  Both directions are bound by memory (the vectors: C * 2 bytes a pixel).
#include "match.h"
#include "match_launch.h"

namespace custma {
namespace {
constexpr int kTW = 64;  // columns of a strip
constexpr int kMaxK = 16;

// rows [y0, y0 + n) x columns [x0, x0 + w) of the image, zeros outside, into LDS
template <typename T>
__device__ __forceinline__ void load_patch_rows(const T* img, int64_t H, int64_t W, int64_t y0, int64_t x0, int n, int w,
                                                float* to) {
    for (int e = threadIdx.x; e < n * w; e += 256) to[e] = ldpad(img, H, W, y0 + e / w, x0 + e % w);
}

template <typename T, typename E>
__global__ __launch_bounds__(256) void k_desc(const T* __restrict__ img, int64_t H, int64_t W, int k, int C8,
                                              ix4* __restrict__ out) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int pw = kTW + k - 1, K = k * k;
    float* tile = (float*)lds;                     // [k][pw]
    float2* stat = (float2*)(tile + ((k * pw + 1) & ~1));  // [64] mean, s
    int* at = (int*)(stat + kTW);                  // [C8] tap -> tile offset, -1 behind the last
    const int64_t strips = cdiv(W, kTW), y = blockIdx.x / strips, x0 = (blockIdx.x % strips) * kTW;
    load_patch_rows(img, H, W, y - k / 2, x0 - k / 2, k, pw, tile);
    for (int t = threadIdx.x; t < C8; t += 256) at[t] = t < K ? t / k * pw + t % k : -1;
    __syncthreads();
    {  // four lanes a pixel
        const int px = threadIdx.x >> 2, part = threadIdx.x & 3;
        const float mid = tile[(k / 2) * pw + px + k / 2];
        float sum = 0.f;
        for (int t = part; t < K; t += 4) sum += tile[at[t] + px] - mid;
        sum += __shfl_xor(sum, 1, 64);
        sum += __shfl_xor(sum, 2, 64);
        const float m = sum / (float)K;
        float ss = 0.f;
        for (int t = part; t < K; t += 4) {
            const float d = (tile[at[t] + px] - mid) - m;
            ss = __builtin_fmaf(d, d, ss);
        }
        ss += __shfl_xor(ss, 1, 64);
        ss += __shfl_xor(ss, 2, 64);
        if (part == 0) stat[px] = make_float2(m, 1.f / sqrtf(ss + kEps));
    }
    __syncthreads();
    const int chunks = C8 / 8;
    const int npx = W - x0 < kTW ? (int)(W - x0) : kTW;
    for (int e = threadIdx.x; e < npx * chunks; e += 256) {
        const int px = e / chunks, c = e % chunks;
        const float2 st = stat[px];
        const float mid = tile[(k / 2) * pw + px + k / 2];
        float v[8];
#pragma unroll
        for (int z = 0; z < 8; ++z) {
            const int o = at[c * 8 + z];
            v[z] = o < 0 ? 0.f : ((tile[o + px] - mid) - st.x) * st.y;
        }
        out[(y * W + x0) * chunks + e] = ix4{pack2<E>(v[0], v[1]), pack2<E>(v[2], v[3]), pack2<E>(v[4], v[5]), pack2<E>(v[6], v[7])};
    }
}

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

template <typename T, typename E>
__global__ __launch_bounds__(256) void k_desc_bwd(const T* __restrict__ img, int64_t H, int64_t W, int k, int C8,
                                                  int band, const ix4* __restrict__ grad, T* __restrict__ out) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int r = k / 2, K = k * k, qw = kTW + k - 1, pw = qw + k - 1, chunks = C8 / 8;
    const int stride = C8 / 2 + 1;                       // dwords per pixel: odd, lanes of a column read apart
    double2* sums = (double2*)lds;                       // [qw] s^2 a, s^2 a m - s b
    float* tile = (float*)(sums + qw);                   // [k][pw] image under the patches of the row
    float* scale = tile + k * pw;                        // [qw] s
    int* gt = (int*)(scale + qw);                        // [qw][stride] gradient vectors of the row
    int16_t* at = (int16_t*)(gt + qw * stride);          // [K] tap -> tile offset
    const int64_t strips = cdiv(W, kTW);
    const int64_t x0 = (blockIdx.x % strips) * kTW, p0 = (blockIdx.x / strips) * band;
    const int64_t p1 = p0 + band < H ? p0 + band : H;
    const int64_t qx0 = x0 - (k - 1) + r;                // first pixel whose patch reaches the strip
    const int64_t ya = p0 - (k - 1) + r < 0 ? 0 : p0 - (k - 1) + r, yb = p1 + r < H ? p1 + r : H;
    const int lane = threadIdx.x & 63, grp = threadIdx.x >> 6;
    for (int t = threadIdx.x; t < K; t += 256) at[t] = (int16_t)(t / k * pw + t % k);
    float acc[kMaxK / 4] = {0.f, 0.f, 0.f, 0.f};         // open image rows P with P % k = grp + 4 e
    const bool inside = x0 + lane < W;

    constexpr int kPre = (kTW + kMaxK - 1) * (kMaxK * kMaxK / 8) / 256 + 1;
    ix4 pre[kPre];
    auto fetch = [&](int64_t y) {
#pragma unroll
        for (int n = 0; n < kPre; ++n) {
            const int e = n * 256 + (int)threadIdx.x;
            pre[n] = ix4{0, 0, 0, 0};
            if (e < qw * chunks && y < yb) {
                const int64_t x = qx0 + e / chunks;
                if (x >= 0 && x < W) pre[n] = grad[(y * W + x) * chunks + e % chunks];
            }
        }
    };
    fetch(ya);
    for (int64_t y = ya; y < yb; ++y) {
        __syncthreads();  // the previous row's readers are done
        load_patch_rows(img, H, W, y - r, qx0 - r, k, pw, tile);
#pragma unroll
        for (int n = 0; n < kPre; ++n) {
            const int e = n * 256 + (int)threadIdx.x;
            if (e < qw * chunks) {
                int* to = gt + e / chunks * stride + e % chunks * 4;
                to[0] = pre[n].x, to[1] = pre[n].y, to[2] = pre[n].z, to[3] = pre[n].w;
            }
        }
        fetch(y + 1);
        __syncthreads();
        const E* g16 = (const E*)gt;
        for (int e = threadIdx.x; e < ((qw * 4 + 63) & ~63); e += 256) {  // four lanes a pixel, whole waves
            const int px = e >> 2 < qw ? e >> 2 : qw - 1, part = e & 3;
            const float mid = tile[r * pw + px + r];
            float sum = 0.f;
            for (int t = part; t < K; t += 4) sum += tile[at[t] + px] - mid;
            sum += __shfl_xor(sum, 1, 64);
            sum += __shfl_xor(sum, 2, 64);
            const float m = sum / (float)K;
            float ss = 0.f, gd = 0.f, gs = 0.f;
            for (int t = part; t < K; t += 4) {
                const float d = (tile[at[t] + px] - mid) - m, gv = (float)g16[px * stride * 2 + t];
                ss = __builtin_fmaf(d, d, ss);
                gd = __builtin_fmaf(d, gv, gd);
                gs += gv;
            }
#pragma unroll
            for (int d = 1; d <= 2; d *= 2) {
                ss += __shfl_xor(ss, d, 64);
                gd += __shfl_xor(gd, d, 64);
                gs += __shfl_xor(gs, d, 64);
            }
            if (part == 0 && e >> 2 < qw) {
                const bool ok = qx0 + px >= 0 && qx0 + px < W;
                const double s = ok ? 1. / sqrt((double)ss + (double)kEps) : 0.;
                const double s2a = s * s * s * (double)gd;  // a = s gd
                scale[px] = (float)s;
                sums[px] = double2{s2a, s2a * ((double)mid + (double)m) - s * (double)gs / (double)K};
            }
        }
        __syncthreads();
        double sa = 0., sb = 0.;
        for (int j = 0; j < k; ++j) {  // patch column j of pixel x0 + lane - j + r
            const double2 v = sums[lane + k - 1 - j];
            sa += v.x;
            sb += v.y;
        }
#pragma unroll
        for (int e = 0; e < kMaxK / 4; ++e) {
            const int slot = grp + 4 * e;
            if (slot >= k) continue;
            // the open row of this slot: P = y - r + i with P % k = slot
            const int64_t low = y - r;
            int i = (int)((slot - low) % k);
            if (i < 0) i += k;
            float s = 0.f;
            for (int j = 0; j < k; ++j) {
                const int q = lane + k - 1 - j;
                s = __builtin_fmaf(scale[q], (float)g16[q * stride * 2 + i * k + j], s);
            }
            // I[P][x0 + lane]: tile row i, tile column of image column x0 + lane is k - 1 + lane
            const double here = (double)tile[i * pw + lane + k - 1];
            acc[e] += (float)((double)s - (here * sa - sb));
            if (i == 0) {  // complete
                if (low >= p0 && low < p1 && inside) out[low * W + x0 + lane] = from_float<T>(acc[e]);
                acc[e] = 0.f;
            }
        }
    }
    // rows that the loop left open: no pixel below the image reaches them
#pragma unroll
    for (int e = 0; e < kMaxK / 4; ++e) {
        const int slot = grp + 4 * e;
        if (slot >= k) continue;
        int i = (int)((slot - (yb - r)) % k);
        if (i < 0) i += k;
        const int64_t P = yb - r + i;
        if (P >= p0 && P < p1 && inside) out[P * W + x0 + lane] = from_float<T>(acc[e]);
    }
}
}  // namespace

int desc_max_kernel() { return kMaxK; }

hipError_t launch_desc(const void* img, int img_dtype, int64_t H, int64_t W, int k, int dtype, void* out, hipStream_t s) {
    const int C8 = (int)cdiv(k * k, 8) * 8, pw = kTW + k - 1;
    const size_t lds = (((size_t)k * pw + 1) & ~(size_t)1) * 4 + kTW * 8 + C8 * 4;
    const dim3 grid((unsigned)(H * cdiv(W, kTW)));
#define CUSTMA_GO(T, E) hipLaunchKernelGGL((k_desc<T, E>), grid, dim3(256), lds, s, (const T*)img, H, W, k, C8, (ix4*)out)
    if (img_dtype == CUSTMA_F16) { if (dtype == CUSTMA_BF16) CUSTMA_GO(__half, __bf16); else CUSTMA_GO(__half, _Float16); }
    else { if (dtype == CUSTMA_BF16) CUSTMA_GO(float, __bf16); else CUSTMA_GO(float, _Float16); }
#undef CUSTMA_GO
    return hipGetLastError();
}

hipError_t launch_desc_bwd(const void* img, int img_dtype, int64_t H, int64_t W, int k, int dtype, const void* grad,
                           void* out, hipStream_t s) {
    const int C8 = (int)cdiv(k * k, 8) * 8, qw = kTW + k - 1, pw = qw + k - 1;
    const size_t lds = (size_t)qw * 16 + (size_t)k * pw * 4 + qw * 4 + (size_t)qw * (C8 / 2 + 1) * 4 + ((k * k * 2 + 3) & ~3);
    const int64_t strips = cdiv(W, kTW);
    // a band re-reads k - 1 rows of its neighbour: bands as tall as leave about four workgroups a compute unit
    int band = 128;
    while (band > 16 && strips * cdiv(H, band) < 1024) band /= 2;
    const dim3 grid((unsigned)(strips * cdiv(H, band)));
#define CUSTMA_GO(T, E) \
    hipLaunchKernelGGL((k_desc_bwd<T, E>), grid, dim3(256), lds, s, (const T*)img, H, W, k, C8, band, (const ix4*)grad, (T*)out)
    if (img_dtype == CUSTMA_F16) { if (dtype == CUSTMA_BF16) CUSTMA_GO(__half, __bf16); else CUSTMA_GO(__half, _Float16); }
    else { if (dtype == CUSTMA_BF16) CUSTMA_GO(float, __bf16); else CUSTMA_GO(float, _Float16); }
#undef CUSTMA_GO
    return hipGetLastError();
}

}  // namespace custma
