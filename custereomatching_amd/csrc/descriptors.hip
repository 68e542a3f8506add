// Patch descriptors: the centred, unit-norm k x k patch of every pixel as a vector of k * k channels, so that
// the dot product of a camera and a projector descriptor is their ZNCC.  Patches as in the cost volume
// (zero-padded, taps at offsets -k/2 .. k-1-k/2), epsilon under the root as there (per vector: ss + 1e-8).
//   x_t = I[p + o_t],  m = mean x,  s = 1 / sqrt(sum (x - m)^2 + eps),  d_t = s (x_t - m)
// Channels are padded with zeros to a multiple of 8 (16 bytes).
//
// Forward.  The mean is separable: per column of the strip the sum of x over k rows, then k of those per pixel, in
// 64 bits, each sum taken anew, not slid from row to row: a pixel that is not finite, or far larger than the rest, stays
// within the patches that hold it.  Means are kept relative to the patch's centre pixel, so that a flat patch gives
// exact zeros.  The squares are summed about the mean, by the lanes that hold the patch anyway: on a high level (0 to
// 255, or 40000) sums of x^2 would cancel, and a flat patch's norm would be their rounding.
//
// Backward.  With a = sum_t g_t d_t and b = mean g,  dI[p] = sum over pixels q whose patch holds p, t = p - q, of
//   s g_t - s b - s^2 a (I[p] - m).
// The last two need only sums over q of s^2 a and of s^2 a m - s b (in 64 bits: around flat patches s is 1e4 and
// they cancel), so every g is read from memory once: on its way to LDS each lane folds its 8 channels into a
// and b.  Over the rows of a patch these sums only ever add (every K rows they are taken back from the last row to
// each of the K, then forward again), so that a value that is not finite, or large, leaves with its row; summing all K
// for each row took 8 % longer on 2048 x 2048, k = 11.  A workgroup walks down a strip of 64 columns; each thread owns a column and every fourth of the k
// image rows that are open at a time, in registers: one owner per sum, no atomics.
//
// The forward is bound by memory (C * 2 bytes a pixel): 2048 x 2048, k = 11 in 227 us, 4.7 TB/s of writes.  The
// backward reads as much in 365 to 440 us: LDS (each 16-bit gradient is read once more per image row that it reaches)
// and three barriers a row.  On a small image it is bound by a workgroup's walk: 330 x 422, k = 15 in 96 us (forward 29).
#include "match.h"
#include "match_launch.h"

namespace custma {
namespace {
constexpr int kTW = 64;  // columns of a strip
constexpr int kMaxK = 16;
// backward: threads and waves of a workgroup (512 measured the same on 330 x 422, 10 % slower on 2048 x 2048)
constexpr int kNT = 256, kGroups = kNT / 64;

__device__ __forceinline__ float load_pixel(const void* img, bool f16, int64_t H, int64_t W, int64_t y, int64_t x) {
    if (y < 0 || y >= H || x < 0 || x >= W) return 0.f;
    return f16 ? __half2float(((const __half*)img)[y * W + x]) : ((const float*)img)[y * W + x];
}
// rows [y0, y0 + n) x columns [x0, x0 + w) of the image, zeros outside, into LDS
__device__ __forceinline__ void load_rows(const void* img, bool f16, int64_t H, int64_t W, int64_t y0, int64_t x0, int n,
                                          int w, float* to) {
    for (int e = threadIdx.x; e < n * w; e += 256) to[e] = load_pixel(img, f16, H, W, y0 + e / w, x0 + e % w);
}

// sum over the LPP consecutive lanes (a power of two up to 32) that the lane belongs to
template <int LPP>
__device__ __forceinline__ float sum_lanes(float v) {
    if constexpr (LPP >= 2) v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xf, 0xf, true));   // lanes ^ 1
    if constexpr (LPP >= 4) v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xf, 0xf, true));   // ^ 2
    if constexpr (LPP >= 8) v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xf, 0xf, true));  // mirrored in 8
    if constexpr (LPP >= 16) v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x140, 0xf, 0xf, true)); // mirrored in 16
    if constexpr (LPP >= 32) v += __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401F));                   // ^ 16
    return v;
}

template <int K>
struct Desc {
    static constexpr int K2 = K * K, CH = (K2 + 7) / 8, C8 = CH * 8;
    static constexpr int LPP = CH <= 1 ? 1 : CH <= 2 ? 2 : CH <= 4 ? 4 : CH <= 8 ? 8 : CH <= 16 ? 16 : 32;  // lanes per pixel
    static constexpr int R = K / 2, QW = kTW + K - 1, PW = QW + K - 1;
    static constexpr int kBand = 16;                  // forward: rows of a workgroup, at most
    static constexpr int STRIDE = C8 / 2 + 1;         // backward: dwords per pixel in LDS, odd
    static constexpr int kFwdLds = (kBand + K - 1) * QW * 4 + kBand * QW * 8 + kBand * kTW * 4;
};

template <typename E, int K>
__global__ __launch_bounds__(256) void k_desc(const void* __restrict__ img, int f16, int64_t H, int64_t W, int band,
                                              ix4* __restrict__ out, float2* __restrict__ stats) {
    using D = Desc<K>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    double* cols = (double*)lds;                            // [band][QW] sums over K rows
    float* mean = (float*)(cols + D::kBand * D::QW);        // [band][64] less the centre pixel
    float* tile = mean + D::kBand * kTW;                    // [band + K - 1][QW]
    const int64_t strips = cdiv(W, kTW), x0 = (blockIdx.x % strips) * kTW, y0 = (blockIdx.x / strips) * band;
    const int rows = H - y0 < band ? (int)(H - y0) : band;
    load_rows(img, f16, H, W, y0 - D::R, x0 - D::R, rows + K - 1, D::QW, tile);
    __syncthreads();
    for (int e = threadIdx.x; e < rows * D::QW; e += 256) {
        const float* from = tile + e;  // row e / QW, column e % QW
        double s1 = 0.;
#pragma unroll
        for (int i = 0; i < K; ++i) s1 += from[i * D::QW];
        cols[e] = s1;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * kTW; e += 256) {
        const int y = e / kTW, x = e % kTW;
        double s1 = 0.;
#pragma unroll
        for (int j = 0; j < K; ++j) s1 += cols[y * D::QW + x + j];
        mean[e] = (float)(s1 / (double)D::K2 - (double)tile[(y + D::R) * D::QW + x + D::R]);
    }
    __syncthreads();
    const int c = threadIdx.x % D::LPP;
    int at[8];
#pragma unroll
    for (int z = 0; z < 8; ++z) at[z] = c * 8 + z < D::K2 ? (c * 8 + z) / K * D::QW + (c * 8 + z) % K : -1;
    for (int e = threadIdx.x / D::LPP; e < rows * kTW; e += 256 / D::LPP) {
        const int y = e / kTW, x = e % kTW;
        if (x0 + x >= W) continue;  // all lanes of the pixel
        const float* from = tile + y * D::QW + x;
        const float m = mean[e], mid = from[D::R * D::QW + D::R];
        float v[8], ss = 0.f;
#pragma unroll
        for (int z = 0; z < 8; ++z) {
            v[z] = at[z] < 0 ? 0.f : (from[at[z] < 0 ? 0 : at[z]] - mid) - m;
            ss = __builtin_fmaf(v[z], v[z], ss);
        }
        ss = sum_lanes<D::LPP>(ss);
        float s = __builtin_amdgcn_rsqf(ss + kEps);
        if (!(ss < INFINITY)) {  // not finite, or beyond 32 bits: in units of 2^80
            ss = 0.f;
#pragma unroll
            for (int z = 0; z < 8; ++z) ss = __builtin_fmaf(v[z] * 0x1p-80f, v[z] * 0x1p-80f, ss);
            s = __builtin_amdgcn_rsqf(sum_lanes<D::LPP>(ss)) * 0x1p-80f;
        }
        const int64_t pixel = (y0 + y) * W + x0 + x;
        if (stats && c == 0) stats[pixel] = make_float2(m, s);
        if (c < D::CH)
            out[pixel * D::CH + c] = ix4{pack2<E>(v[0] * s, v[1] * s), pack2<E>(v[2] * s, v[3] * s),
                                         pack2<E>(v[4] * s, v[5] * s), pack2<E>(v[6] * s, v[7] * s)};
    }
}

template <typename E, int K>
__global__ __launch_bounds__(kNT) void k_desc_bwd(const void* __restrict__ img, int f16, int64_t H, int64_t W, int band,
                                                  const float2* __restrict__ stats, const ix4* __restrict__ grad,
                                                  const float* __restrict__ factor, void* __restrict__ out) {
    using D = Desc<K>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    double2* past = (double2*)lds;                       // [K][QW] s^2 a, s^2 a m - s b of rows of pixels
    double2* sums = past + K * D::QW;                    // [QW] the last K rows' sums
    float* scale = (float*)(sums + D::QW);               // [QW] s
    int* gt = (int*)(scale + D::QW);                     // [QW][STRIDE] gradient vectors of a row of pixels
    float* ring = (float*)(gt + D::QW * D::STRIDE);      // [2 K][PW] image rows, each twice K apart: K in a row at any time
    const int64_t strips = cdiv(W, kTW);
    const int64_t x0 = (blockIdx.x % strips) * kTW, p0 = (blockIdx.x / strips) * band;
    const int64_t p1 = p0 + band < H ? p0 + band : H;
    const int64_t qx0 = x0 - (K - 1) + D::R;             // first pixel whose patch reaches the strip
    const int64_t yt = p0 - (K - 1) + D::R;              // and its row
    const int64_t ya = yt < 0 ? 0 : yt, yb = p1 + D::R < H ? p1 + D::R : H;
    const int lane = threadIdx.x & 63, grp = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // LPP lanes a pixel, 8 channels each, PPI pixels at a time
    constexpr int PPI = kNT / D::LPP, ITER = (D::QW + PPI - 1) / PPI;
    static_assert(ITER <= D::LPP, "one lane of a pixel's group per pass");
    const int c = threadIdx.x % D::LPP, first = threadIdx.x / D::LPP;
    int at[8], keep[4];                                  // tap offsets; channels behind the last tap are masked out
#pragma unroll
    for (int z = 0; z < 8; ++z) at[z] = c * 8 + z < D::K2 ? (c * 8 + z) / K * D::PW + (c * 8 + z) % K : 0;
#pragma unroll
    for (int z = 0; z < 4; ++z)
        keep[z] = (c * 8 + 2 * z < D::K2 ? 0xffff : 0) | (c * 8 + 2 * z + 1 < D::K2 ? (int)0xffff0000 : 0);
    // the pixel whose sums this lane finishes
    const int mine = c * PPI + first;
    const bool finish = c < ITER && mine < D::QW, mine_in = finish && qx0 + mine >= 0 && qx0 + mine < W;

    // A row of pixels' gradients and statistics, and the image row that it adds.  Addresses are clamped into the
    // arrays and what they should not have read is zeroed where it is used: a load under a condition would be
    // waited for on the spot.
    ix4 pre[ITER];
    float2 st;
    uint32_t pix;
    const int cl = c < D::CH ? c : D::CH - 1;
    auto fetch = [&](int64_t y) {
        const int64_t yr = y < yb ? y : yb - 1;
#pragma unroll
        for (int n = 0; n < ITER; ++n) {
            int64_t x = qx0 + n * PPI + first;
            x = x < 0 ? 0 : x < W ? x : W - 1;
            pre[n] = grad[(yr * W + x) * D::CH + cl];
        }
        st = stats[yr * W + (mine_in ? qx0 + mine : 0)];
        int64_t py = y - D::R + K - 1, px = qx0 - D::R + threadIdx.x;
        py = py < 0 ? 0 : py < H ? py : H - 1;
        px = px < 0 ? 0 : px < W ? px : W - 1;
        if (f16) pix = ((const uint16_t*)img)[py * W + px];
        else pix = ((const uint32_t*)img)[py * W + px];
    };
    constexpr int SLOTS = (K + kGroups - 1) / kGroups;
    float acc[SLOTS];                                    // sum s g of the open image rows P with P % K = grp + kGroups e
#pragma unroll
    for (int e = 0; e < SLOTS; ++e) acc[e] = 0.f;
    double va = 0., vb = 0.;
    const bool inside = x0 + lane < W;
    const float times = factor ? factor[0] : 1.f;
    auto put = [&](int64_t P, float v) {
        v *= times;
        if (P < p0 || P >= p1 || !inside) return;
        if (f16) ((__half*)out)[P * W + x0 + lane] = __float2half_rn(v);
        else ((float*)out)[P * W + x0 + lane] = v;
    };

    int slot0 = 0;                                       // ring slot of the first row of the present patches
    fetch(ya);
    for (int e = threadIdx.x; e < (K - 1) * D::PW; e += kNT) {
        const float v = load_pixel(img, f16, H, W, ya - D::R + e / D::PW, qx0 - D::R + e % D::PW);
        ring[e] = v;
        ring[K * D::PW + e] = v;
    }
    for (int e = threadIdx.x; e < K * D::QW; e += kNT) past[e] = double2{0., 0.};
    int base = (int)(((ya - D::R) % K + K) % K);         // slot of the image row that closes with row y of pixels
    // rows behind the last pixel row run too, without pixels, until the strip's image rows are closed
    for (int64_t y = ya; y < p1 + D::R; ++y) {
        const bool any = y < yb;
        const int in = slot0 + K - 1 < K ? slot0 + K - 1 : slot0 - 1;
        if (threadIdx.x < D::PW) {
            const int64_t py = y - D::R + K - 1, px = qx0 - D::R + threadIdx.x;
            float v = f16 ? __half2float(__ushort_as_half((unsigned short)pix)) : __builtin_bit_cast(float, pix);
            if (py >= H || px < 0 || px >= W) v = 0.f;   // py >= 0: the first K - 1 rows were loaded ahead
            ring[in * D::PW + threadIdx.x] = v;
            ring[(in + K) * D::PW + threadIdx.x] = v;
        }
        ix4 cur[ITER];
#pragma unroll
        for (int n = 0; n < ITER; ++n) {
            const int px = n * PPI + first;
            const bool ok = any && c < D::CH && qx0 + px >= 0 && qx0 + px < W;
#pragma unroll
            for (int z = 0; z < 4; ++z) cur[n][z] = ok ? pre[n][z] & keep[z] : 0;
            if (px < D::QW && c < D::CH) {
                int* to = gt + px * D::STRIDE + c * 4;
                to[0] = cur[n].x, to[1] = cur[n].y, to[2] = cur[n].z, to[3] = cur[n].w;
            }
        }
        const float2 cst = st;
        fetch(y + 1);
        __syncthreads();
        const float* rows = ring + slot0 * D::PW;        // the row's patches
        float gd = 0.f, gs = 0.f;
#pragma unroll
        for (int n = 0; n < ITER; ++n) {
            const int px = n * PPI + first, pc = px < D::QW ? px : D::QW - 1;
            const float* from = rows + pc;
            const float mid = from[D::R * D::PW + D::R];
            float d = 0.f, s = 0.f;
#pragma unroll
            for (int z = 0; z < 8; ++z) {
                const fx2 g2 = unpack2<E>(cur[n][z / 2]);
                const float g = z & 1 ? g2.y : g2.x;
                d = __builtin_fmaf(from[at[z]] - mid, g, d);
                s += g;
            }
            d = sum_lanes<D::LPP>(d);
            s = sum_lanes<D::LPP>(s);
            if (c == n) gd = d, gs = s;
        }
        if (finish) {
            double s = 0.;                               // a pixel outside adds nothing
            double2 now = {0., 0.};
            if (any && mine_in) {
                s = cst.y;
                const double m = cst.x, mid = rows[D::R * D::PW + D::R + mine];
                now.x = s * s * s * ((double)gd - m * (double)gs);  // s^2 a, a = s sum g (x - mean)
                now.y = now.x * (mid + m) - s * (double)gs * (1. / (double)D::K2);
            }
            // of the last K rows: those since slot 0 in va, vb, those before it in the sums from each slot to the last
            va += now.x;
            vb += now.y;
            double2 all = {va, vb};
            if (slot0 + 1 < K) {
                const double2 v = past[(slot0 + 1) * D::QW + mine];
                all.x += v.x;
                all.y += v.y;
            }
            past[slot0 * D::QW + mine] = now;
            if (slot0 + 1 == K) {
                double2 v = now;
#pragma unroll
                for (int i = K - 2; i >= 0; --i) {
                    const double2 u = past[i * D::QW + mine];
                    v.x += u.x;
                    v.y += u.y;
                    past[i * D::QW + mine] = v;
                }
                va = vb = 0.;
            }
            scale[mine] = (float)s;
            sums[mine] = all;
        }
        __syncthreads();
        const int64_t low = y - D::R;  // the image row that closes with this row of pixels
        float sc[K];
#pragma unroll
        for (int j = 0; j < K; ++j) sc[j] = scale[lane + K - 1 - j];  // patch column j: pixel x0 + lane - j + R
#pragma unroll
        for (int e = 0; e < SLOTS; ++e) {
            const int slot = grp + kGroups * e;
            if (slot >= K) continue;
            int i = slot - base;  // the open row of this slot is low + i
            if (i < 0) i += K;
            if (low + i < p0 || low + i >= p1) continue;
            const E* g16 = (const E*)(gt + (lane + K - 1) * D::STRIDE) + i * K;
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < K; ++j) s = __builtin_fmaf(sc[j], (float)g16[j - j * D::STRIDE * 2], s);
            acc[e] += s;
            if (i == 0) {
                double sa = 0., sb = 0.;
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    const double2 v = sums[lane + K - 1 - j];
                    sa += v.x;
                    sb += v.y;
                }
                const double here = (double)rows[lane + K - 1];
                put(low, (float)((double)acc[e] - (here * sa - sb)));
                acc[e] = 0.f;
            }
        }
        slot0 = slot0 + 1 < K ? slot0 + 1 : 0;
        base = base + 1 < K ? base + 1 : 0;
        __syncthreads();
    }
}

template <typename E, int K>
hipError_t go_fwd(const void* img, bool f16, int64_t H, int64_t W, void* out, float2* stats, hipStream_t s) {
    int band = Desc<K>::kBand;
    while (band > 4 && cdiv(W, kTW) * cdiv(H, band) < 1024) band /= 2;
    hipLaunchKernelGGL((k_desc<E, K>), dim3((unsigned)(cdiv(W, kTW) * cdiv(H, band))), dim3(256), Desc<K>::kFwdLds, s, img,
                       (int)f16, H, W, band, (ix4*)out, stats);
    return hipGetLastError();
}
template <typename E, int K>
hipError_t go_bwd(const void* img, bool f16, int64_t H, int64_t W, const float2* stats, const void* grad,
                  const float* factor, void* out, hipStream_t s) {
    using D = Desc<K>;
    const int lds = (K + 1) * D::QW * 16 + D::QW * 4 + D::QW * D::STRIDE * 4 + 2 * K * D::PW * 4;
    // a band re-reads K - 1 rows of its neighbour and walks them: as few bands as fill the chip once (at least 4 rows
    // each: 94 us against 105 with 8 on 330 x 422, k = 15)
    const int64_t slots = 256 * (163840 / lds < 4 ? 163840 / lds : 4), strips = cdiv(W, kTW);
    const int64_t rows = cdiv(H, slots / strips > 0 ? slots / strips : 1);
    const int band = (int)(rows < 4 ? 4 : rows > 128 ? 128 : rows);
    auto fn = k_desc_bwd<E, K>;
    static std::atomic<uint64_t> lds_done{0};
    const hipError_t e = allow_lds((const void*)fn, lds, lds_done);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(fn, dim3((unsigned)(strips * cdiv(H, band))), dim3(kNT), lds, s, img, (int)f16, H, W, band,
                       stats, (const ix4*)grad, factor, out);
    return hipGetLastError();
}

template <typename E, int K = 1>
hipError_t by_k(int k, bool bwd, const void* img, bool f16, int64_t H, int64_t W, void* out, float2* stats,
                const void* grad, const float* factor, hipStream_t s) {
    if constexpr (K > kMaxK) {
        return hipErrorInvalidValue;
    } else {
        if (k != K) return by_k<E, K + 1>(k, bwd, img, f16, H, W, out, stats, grad, factor, s);
        return bwd ? go_bwd<E, K>(img, f16, H, W, stats, grad, factor, out, s) : go_fwd<E, K>(img, f16, H, W, out, stats, s);
    }
}
}  // namespace

int desc_max_kernel() { return kMaxK; }

hipError_t launch_desc(const void* img, int img_dtype, int64_t H, int64_t W, int k, int dtype, void* out, float* stats,
                       hipStream_t s) {
    const bool f16 = img_dtype == CUSTMA_F16;
    return dtype == CUSTMA_BF16 ? by_k<__bf16>(k, false, img, f16, H, W, out, (float2*)stats, nullptr, nullptr, s)
                                : by_k<_Float16>(k, false, img, f16, H, W, out, (float2*)stats, nullptr, nullptr, s);
}
hipError_t launch_desc_bwd(const void* img, int img_dtype, int64_t H, int64_t W, int k, int dtype, const float* stats,
                           const void* grad, const float* factor, void* out, hipStream_t s) {
    const bool f16 = img_dtype == CUSTMA_F16;
    return dtype == CUSTMA_BF16 ? by_k<__bf16>(k, true, img, f16, H, W, out, (float2*)stats, grad, factor, s)
                                : by_k<_Float16>(k, true, img, f16, H, W, out, (float2*)stats, grad, factor, s);
}

}  // namespace custma
