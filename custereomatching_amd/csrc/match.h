// Row matching on vectors: softmax read-out (attention) and softmax cross entropy between the positions
// of two rows, on vectors per pixel instead of raw patches.  Shared by match_fwd.hip, match_bwd.hip and
// match_wide.hip.
//
// Scores.  Query i of batch entry b and head h sits at position p = offset_b + i; key j is visible to it iff
//   j < length_b,  j <= p + right,  and  (j >= p - left or j < sinks)
// (a bound that is -1 does not hold).  Per query this is [0, min(sinks, hi)) + [lo, hi) with
//   hi = clamp(p + right + 1, 0, length),  lo = clamp(p - left, 0, hi).
//
// Rows.  The G query heads that share a key head are packed into one row axis, r = i * G + g, so that a
// key tile is read once for the whole group and the gradients of a shared head sum inside the kernel.
//
// Matrix instruction.  v_mfma_f32_32x32x16: lane l holds column l % 32 of B and row l % 32 of A, eight
// contraction slots 8 * (l / 32) ..; its result holds column l % 32 and rows 8 * (t / 4) + 4 * (l / 32) + t % 4,
// t = 0 .. 15.  Scores are computed transposed (A = keys, B = queries): a lane then holds one query's
// scores, the softmax needs one exchange between the wave's halves, and the result registers are already
// the B operand of the next product if its contraction slots are numbered
//   slot s of half h in step u  ->  key 16 u + 8 * (s / 4) + 4 h + s % 4,
// which the other operand follows by reading LDS with the transposing ds_read (4 rows x 16 columns per
// 16 lanes).  No value crosses lanes between the two products.
//
// LDS tiles are [rows][channels] of 16-bit elements, filled 16 bytes a lane straight from memory
// (global_load_lds).  Chunk c (16 bytes) of row r sits at position c ^ swz(r): 8 lanes that read one
// chunk of 8 consecutive rows, and the 4 rows x 32 bytes of a transposing read, then fall into different banks.
#pragma once
#include <hip/hip_bf16.h>

#include "common.h"

namespace custma {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kMatchMaxC = 256;  // channels the row kernels hold in registers; wider: match_wide.hip

struct MatchGeo {
    int64_t qs[3], ks[3], vs[3];  // element strides: batch, position, head
    const int32_t* offset;        // [B] position of the first query (null: 0)
    const int32_t* length;        // [B] keys in use (null: Lk)
    int32_t B, Lq, Lk, Hkv, G, C, Cv;
    int32_t sinks;
    int64_t left, right;          // -1: no bound
    float scale;
    __host__ __device__ int32_t rows() const { return Lq * G; }
    __host__ __device__ int64_t heads() const { return (int64_t)Hkv * G; }
};

struct Span {
    int32_t lo, hi;
};

__device__ __forceinline__ int32_t key_length(const MatchGeo& g, int b) {
    if (!g.length) return g.Lk;
    const int32_t n = g.length[b];
    return n < 0 ? 0 : n > g.Lk ? g.Lk : n;
}

__device__ __forceinline__ Span span_of(const MatchGeo& g, int64_t off, int32_t len, int32_t i) {
    const int64_t p = off + i;
    Span s;
    s.hi = len;
    if (g.right >= 0) {
        const int64_t e = p + g.right + 1;
        s.hi = e < 0 ? 0 : e < len ? (int32_t)e : len;
    }
    s.lo = 0;
    if (g.left >= 0) {
        const int64_t a = p - g.left;
        s.lo = a < 0 ? 0 : a < s.hi ? (int32_t)a : s.hi;
    }
    return s;
}

// ---- 16-bit element types ----
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef float fx2 __attribute__((ext_vector_type(2)));
typedef float fx16 __attribute__((ext_vector_type(16)));
typedef int ix4 __attribute__((ext_vector_type(4)));
typedef int ix2 __attribute__((ext_vector_type(2)));
typedef short sx4 __attribute__((ext_vector_type(4)));

template <typename E>
struct Half16;
template <>
struct Half16<_Float16> {
    typedef f16x8 x8;
    typedef f16x2 x2;
    // 2^e that keeps probabilities down to 2^-28 normal in the gradient products (their weights are <= 1)
    static constexpr float kLift = 14.f;
    static __device__ __forceinline__ fx16 mma(ix4 a, ix4 b, fx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
    }
};
template <>
struct Half16<__bf16> {
    typedef b16x8 x8;
    typedef b16x2 x2;
    static constexpr float kLift = 0.f;
    static __device__ __forceinline__ fx16 mma(ix4 a, ix4 b, fx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
    }
};

template <typename E>
__device__ __forceinline__ int pack2(float a, float b) {  // round to nearest even
    const fx2 v = {a, b};
    return __builtin_bit_cast(int, __builtin_convertvector(v, typename Half16<E>::x2));
}
template <typename E>
__device__ __forceinline__ fx2 unpack2(int v) {
    return __builtin_convertvector(__builtin_bit_cast(typename Half16<E>::x2, v), fx2);
}

// ---- LDS tiles ----
typedef __attribute__((address_space(3))) char lds_char;

template <int NCH>
__device__ __forceinline__ int swz(int row) {
    constexpr int rpl = NCH >= 16 ? 1 : 16 / NCH;  // rows per 256 bytes of LDS
    constexpr int mask = (NCH < 16 ? NCH : 16) - 1;
    return (row / rpl) & mask;
}

// 16 zero bytes in memory: what rows and channels behind the end are filled from
static __device__ __attribute__((aligned(16))) const int kZeros[4] = {0, 0, 0, 0};

// 16 bytes per lane from memory to LDS, lane l's behind `to` + 16 l.  Inline asm: the compiler's own counting
// cannot tell one LDS buffer from the other and would wait for the tile in flight before reading the present
// one.  The load writes no register; wait_fills() and a barrier stand between it and the tile's readers.
__device__ __forceinline__ void load_lds16(const char* src, char* to) {
    const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)to;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(at)), "v"((uint64_t)(uintptr_t)src)
                 : "memory");
}
// Fill a [ROWS][NCH * 8] tile from the row addresses row(t) (null: zeros), zeros behind `chunks` 16-byte
// chunks.  All of the block's NW waves take part.
template <int ROWS, int NCH, int NW, typename Row>
__device__ __forceinline__ void fill_rows(char* tile, Row row_at, int chunks, int wave, int lane) {
    constexpr int total = ROWS * NCH;
    static_assert(total % 64 == 0, "whole loads");
#pragma unroll
    for (int n = 0; n < (total + NW * 64 - 1) / (NW * 64); ++n) {
        const int id = (n * NW + wave) * 64;  // uniform: first chunk of this load
        if (total % (NW * 64) != 0 && id >= total) break;
        const int row = (id + lane) / NCH, c = ((id + lane) % NCH) ^ swz<NCH>(row);
        const char* src = row_at(row);
        src = src && c < chunks ? src + c * 16 : (const char*)kZeros;
        load_lds16(src, tile + id * 16);
    }
}
// the same where row t is memory row first + t, stride bytes apart, while first + t < end
template <int ROWS, int NCH, int NW>
__device__ __forceinline__ void fill_tile(char* tile, const char* base, int64_t stride, int first, int end,
                                          int chunks, int wave, int lane) {
    fill_rows<ROWS, NCH, NW>(
        tile, [&](int t) { return first + t < end ? base + (int64_t)(first + t) * stride : nullptr; }, chunks, wave, lane);
}
__device__ __forceinline__ void wait_fills() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// A / B operand from a tile whose rows are the operand's rows: lane l reads 8 elements of row0 + l % 32
template <int NCH>
__device__ __forceinline__ ix4 frag_rows(const char* tile, int row0, int step, int lane) {
    const int row = lane & 31;
    const int at = (row * NCH + ((lane >> 5) ^ swz<NCH>(row))) * 16;
    return *(const ix4*)(tile + row0 * NCH * 16 + (at ^ (step * 32)));
}
// transposed operand: lane l gets column col0 + l % 32 of the 16 rows row0 .. row0 + 15, rows numbered as
// 8 * (s / 4) + 4 h + s % 4 (see the head of this file); row0 a multiple of 16, col0 of 32
template <int NCH>
__device__ __forceinline__ ix4 frag_cols(const char* tile, int row0, int col0, int lane) {
    const int x = lane & 15, row = 4 * (lane >> 5) + (x >> 2);
    const int chunk = 2 * ((lane >> 4) & 1) + ((x & 3) >> 1);
    const int at = (row * NCH + (chunk ^ swz<NCH>(row))) * 16 + (x & 1) * 8;
    const int flip = (col0 / 8) * 16;
    const char* t = tile + row0 * NCH * 16;
    const sx4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) sx4*)(t + (at ^ flip)));
    const sx4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) sx4*)(t + 8 * NCH * 16 + (at ^ flip ^ (swz<NCH>(8) * 16))));
    const ix2 lo = __builtin_bit_cast(ix2, a), hi = __builtin_bit_cast(ix2, b);
    return ix4{lo.x, lo.y, hi.x, hi.y};
}

// the same with the rows in their own order, 8 h + s: what frag_rows of the other operand goes with
template <int NCH>
__device__ __forceinline__ ix4 frag_cols_plain(const char* tile, int row0, int col0, int lane) {
    const int x = lane & 15, row = 8 * (lane >> 5) + (x >> 2);
    const int chunk = 2 * ((lane >> 4) & 1) + ((x & 3) >> 1);
    const int at = (row * NCH + (chunk ^ swz<NCH>(row))) * 16 + (x & 1) * 8;
    const int flip = (col0 / 8) * 16;
    const char* t = tile + row0 * NCH * 16;
    const sx4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) sx4*)(t + (at ^ flip)));
    const sx4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) sx4*)(t + 4 * NCH * 16 + (at ^ flip ^ (swz<NCH>(4) * 16))));
    const ix2 lo = __builtin_bit_cast(ix2, a), hi = __builtin_bit_cast(ix2, b);
    return ix4{lo.x, lo.y, hi.x, hi.y};
}

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace custma
