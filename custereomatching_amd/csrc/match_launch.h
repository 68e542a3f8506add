// Host side of the matching operators: what the launchers of match_*.hip and descriptors.hip take.
#pragma once
#include <atomic>

#include "match.h"

namespace custma {

// What a forward writes.  With more than one split of the keys: part [split][row][Cv] (unnormalised),
// part_ml [split][row][4] (maximum and sum in base 2, target's score), then joined by launch_match_join.
struct FwdOut {
    void* out;              // [B, Lq, heads, Cv]
    void* low;              // null, or the 16-bit output's rounding error, also in 16 bits
    float* lse;             // [B, Lq, heads]
    float* loss;            // cross entropy: [B, Lq]
    const int64_t* target;  // cross entropy: [B, Lq]
    float* part;
    float* part_ml;
};

inline int pad_channels(int c) { return c <= 32 ? 32 : c <= 64 ? 64 : c <= 128 ? 128 : 256; }

// LDS above 64 KiB has to be allowed for each kernel, on each device, once.  `done`: a bit per device, one word a kernel
// (devices past 64 ask again on every call).
inline hipError_t allow_lds(const void* fn, int bytes, std::atomic<uint64_t>& done) {
    if (bytes <= 65536) return hipSuccess;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return hipSuccess;
    e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

#define CUSTMA_MATCH_DECL(HD)                                                                                         \
    hipError_t launch_match_fwd_##HD(const MatchGeo& g, int dtype, bool wide_out, bool few, int hdv, const void* q,   \
                                     const void* k, const void* v, const FwdOut& o, int nsplit, hipStream_t s);       \
    hipError_t launch_match_bwd_q_##HD(const MatchGeo& g, int dtype, int hdv, const BwdArgs& a, hipStream_t s);       \
    hipError_t launch_match_bwd_k_##HD(const MatchGeo& g, int dtype, int hdv, const BwdArgs& a, bool sinks,           \
                                       int nsplit, hipStream_t s);

// What the backward kernels read and write.  Attention: go is the 16-bit output gradient [B, Lq, heads, Cv].
// Cross entropy (hdv = 0): go is not used.  Results are multiplied by *factor (null: 1) and by scale (grad_v by
// *factor only).
struct BwdArgs {
    const void *q, *k, *v, *go;
    // per packed row, [B][Hkv][rows] each (launch_match_rows): what the score's product starts from, kLift - lse in base
    // 2 over the score's factor (-inf for a row that does not count); what dP starts from, minus go . out (cross
    // entropy: the row's weight); cross entropy: its target, -1 where it does not count
    float *start, *second;
    int32_t *hot;
    const float *lse;      // cross entropy, wide vectors
    const int64_t* target;
    const float* weight;   // below 2 in size; null: 1 for every counted row
    const float* factor;
    void *gq, *gk, *gv;    // 16-bit, contiguous; gv may be null
    float *part_k, *part_v;  // 32-bit [split][B][keys][Hkv][C / Cv]: partial sums over row splits, before factor and scale
    const float *init_k, *init_v;  // [B][init_keys][Hkv][C / Cv]: what the sinks' own pass found, added in
    int32_t init_keys;
};
CUSTMA_MATCH_DECL(32)
CUSTMA_MATCH_DECL(64)
CUSTMA_MATCH_DECL(128)
CUSTMA_MATCH_DECL(256)

hipError_t launch_match_join(const MatchGeo& g, int dtype, bool wide_out, const FwdOut& o, int nsplit, hipStream_t s);
// out16 = go (32-bit) times a power of two near 1 / max |go|, scale[0] = its inverse; partials: 1024 floats
hipError_t launch_match_narrow(const float* go, int64_t n, int dtype, void* out16, float* scale, float* partials,
                               hipStream_t s);
// out = weight times a power of two, the largest in [1, 2); scale[0] = factor (null: 1) over that power.  weight may be
// null (scale only); partials: 1024 floats
hipError_t launch_match_weights(const float* weight, int64_t n, const float* factor, float* out, float* scale,
                                float* partials, hipStream_t s);
// fills a.start, a.second, a.hot; attention (out given): go . out with out + low of the forward
hipError_t launch_match_rows(const MatchGeo& g, int dtype, const BwdArgs& a, const float* lse, const void* out,
                             bool out_f32, const void* low, hipStream_t s);
// sums over row splits of n and n2 values (an `out` may be null) -> 16-bit gradients times factor and scale, or 32-bit
// sums where `to32`
hipError_t launch_match_sum(const float* part, int nsplit, int64_t n, int dtype, bool to32, const float* factor,
                            float scale, void* out, const float* part2, int64_t n2, float scale2, void* out2, hipStream_t s);
// total[0] = sum of loss over counted rows, total[1] = 1 / max(1, count); partials: 2 * 1024 doubles
hipError_t launch_match_total(const float* loss, const int64_t* target, const MatchGeo& g, int64_t n, float* total,
                              double* partials, hipStream_t s);

// stats (null or 2 floats a pixel): mean less the centre pixel, 1 / norm; what the backward takes.  The image gradient
// is multiplied by *factor (null: 1).
hipError_t launch_desc(const void* img, int img_dtype, int64_t H, int64_t W, int k, int dtype, void* out, float* stats,
                       hipStream_t s);
hipError_t launch_desc_bwd(const void* img, int img_dtype, int64_t H, int64_t W, int k, int dtype, const float* stats,
                           const void* grad, const float* factor, void* out, hipStream_t s);
int desc_max_kernel();

// Wide vectors (match_wide.hip), no bounds: forward over `nsplit` ranges of the classes, two parts each, parts
// [2 nsplit][rows][4] as in FwdOut::part_ml; backward in pieces of the classes.
int wide_splits(const MatchGeo& g);
hipError_t launch_wide_fwd(const MatchGeo& g, int dtype, const void* q, const void* k, const FwdOut& o, hipStream_t s);
size_t wide_bwd_bytes(const MatchGeo& g);
hipError_t launch_wide_bwd(const MatchGeo& g, int dtype, const BwdArgs& a, void* ws, hipStream_t s);

}  // namespace custma
