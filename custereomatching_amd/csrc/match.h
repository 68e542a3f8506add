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
// (global_load_lds).  Chunk c (16 bytes) of row r sits at position c ^ swz(r), so that 8 lanes that read one
// chunk of 8 consecutive rows fall into different banks, and so do the 4 rows x 64 bytes that 32 lanes of a
// transposing read ask for (rows that share a 256-byte line of banks differ in which quarter of it they use).
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
    int32_t left, right, sinks;   // -1: no bound
    float scale;
    __host__ __device__ int32_t rows() const { return Lq * G; }
    __host__ __device__ int64_t heads() const { return (int64_t)Hkv * G; }
};

// xcd_remap in 32 bits: a 64-bit division costs a workgroup of these kernels more than a tile
__device__ __forceinline__ uint32_t xcd_block() {
    const uint32_t b = blockIdx.x, n = gridDim.x, q = n / 8, rem = n % 8, x = b % 8, i = b / 8;
    return x < rem ? x * (q + 1) + i : rem * (q + 1) + (x - rem) * q + i;
}
// quotient and remainder of uniform values, kept uniform (the division itself runs in vector registers)
__device__ __forceinline__ uint32_t split_off(uint32_t& id, uint32_t n) {
    if (n == 1) return 0;
    const uint32_t q = id / n, r = id - q * n;
    id = __builtin_amdgcn_readfirstlane(q);
    return __builtin_amdgcn_readfirstlane(r);
}
// part s of n of `tiles` (below 2^25, n at most 64)
__device__ __forceinline__ int part_of(int tiles, int s, int n) {
    return n == 1 ? s * tiles : (int)((uint32_t)tiles * (uint32_t)s / (uint32_t)n);
}

struct Span {
    int32_t lo, hi;
};

__device__ __forceinline__ int32_t key_length(const MatchGeo& g, int b) {
    if (!g.length) return g.Lk;
    const int32_t n = g.length[b];
    return n < 0 ? 0 : n > g.Lk ? g.Lk : n;
}
constexpr int32_t kMaxPos = 1 << 30;  // of offsets: positions off + i then fit in 32 bits
__device__ __forceinline__ int32_t first_position(const MatchGeo& g, int b) {
    if (!g.offset) return 0;
    const int32_t o = g.offset[b];
    return o < -kMaxPos ? -kMaxPos : o > kMaxPos ? kMaxPos : o;
}
__device__ __forceinline__ int32_t position_of_row(const MatchGeo& g, int32_t r) { return g.G == 1 ? r : r / g.G; }

__device__ __forceinline__ Span span_of(const MatchGeo& g, int32_t off, int32_t len, int32_t i) {
    const int32_t p = off + i;  // [-2^30, 2^31), and each bound below 2^31: no sum here leaves 32 bits
    Span s;
    s.hi = len;
    if (g.right >= 0 && p < len && g.right < len - 1 - p) {
        const int32_t e = p + g.right + 1;
        s.hi = e < 0 ? 0 : e;
    }
    s.lo = 0;
    if (g.left >= 0) {
        const int32_t a = (p < 0 ? 0 : p) - g.left;
        s.lo = a < 0 ? 0 : a < s.hi ? a : s.hi;
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
__device__ __forceinline__ constexpr int swz(int row) {
    return NCH >= 16 ? (row & 3) * 4 | (row >> 2 & 3) : NCH == 8 ? (row >> 1 & 1) * 4 | (row >> 2 & 3) : row >> 2 & 3;
}
__device__ __forceinline__ uint32_t lds_offset(const char* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

// 16 zero bytes in memory: what rows and channels behind the end are filled from
static __device__ __attribute__((aligned(16))) const int kZeros[4] = {0, 0, 0, 0};

// 16 bytes per lane from memory to LDS, lane l's behind `to` + 16 l.  Inline asm: the compiler's own counting
// cannot tell one LDS buffer from the other and would wait for the tile in flight before reading the present
// one.  The load writes no register; wait_fills() and a barrier stand between it and the tile's readers.  The compiler
// does not see into the asm, so the wait states are in it: one between m0 and the load, and five where the load's address
// is in scalar registers, which a vector instruction (v_readfirstlane, or v_readlane of a spilled one) may have written
// just before (hazard_check.py verifies the five on the code of every build).
__device__ __forceinline__ void load_lds16(const char* src, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(to)), "v"((uint64_t)(uintptr_t)src)
                 : "memory", "m0");
}
__device__ __forceinline__ uint64_t uniform64(const char* p) {
    const uint64_t v = (uint64_t)(uintptr_t)p;
    return (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v);
}
// the same from a uniform address and a 32-bit offset per lane
__device__ __forceinline__ void load_lds16(const char* base, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(to)), "v"(offset), "s"(uniform64(base))
                 : "memory", "m0");
}
// Fills [ROWS][NCH * 8] tiles, all of the block's NW waves taking part.  Where a lane reads within a tile does not
// change from tile to tile (`off`, set up once by init from the byte offset of a row); a tile costs the uniform
// address of its first row.  Chunks behind the vectors' own are never written (clear_tails).
template <int ROWS, int NCH, int NW>
struct Filler {
    static constexpr int total = ROWS * NCH, N = (total + NW * 64 - 1) / (NW * 64);
    static_assert(total % 64 == 0, "whole loads");
    static constexpr uint32_t kNothing = ~0u;  // the lane's chunk is behind the vectors' own
    uint32_t off[N];
    int chunks, wave, lane;
    __device__ __forceinline__ int id(int n) const { return (n * NW + wave) * 64; }  // uniform: first chunk of load n
    __device__ __forceinline__ int row(int n) const { return (id(n) + lane) / NCH; }
    __device__ __forceinline__ int chunk(int n) const { return ((id(n) + lane) % NCH) ^ swz<NCH>(row(n)); }
    template <typename Row>
    __device__ __forceinline__ void init(int chunks_, int wave_, int lane_, Row row_offset) {
        chunks = chunks_, wave = wave_, lane = lane_;
#pragma unroll
        for (int n = 0; n < N; ++n) off[n] = chunk(n) < chunks ? row_offset(row(n)) + chunk(n) * 16 : kNothing;
    }
    // rows [0, valid) of the tile whose row 0 is at base; those behind it repeat the last one (they are masked)
    template <typename Row>
    __device__ __forceinline__ void fill(uint32_t tile, const char* base, int valid, Row row_offset) const {
        if (valid >= ROWS) {
            if (chunks == NCH) {
#pragma unroll
                for (int n = 0; n < N; ++n)
                    if (total % (NW * 64) == 0 || id(n) < total) load_lds16(base, off[n], tile + id(n) * 16);
            } else {
#pragma unroll
                for (int n = 0; n < N; ++n)
                    if ((total % (NW * 64) == 0 || id(n) < total) && off[n] != kNothing)
                        load_lds16(base, off[n], tile + id(n) * 16);
            }
        } else {
#pragma unroll 1
            for (int n = 0; n < N; ++n) {
                if (total % (NW * 64) != 0 && id(n) >= total) break;
                const uint32_t o = row_offset(row(n) < valid ? row(n) : valid - 1) + chunk(n) * 16;
                if (chunk(n) < chunks) load_lds16(base, o, tile + id(n) * 16);
            }
        }
    }
};
// A place in the walk over key tiles: the sinks in front of the window, then the window.
struct KeyWalk {
    int tile, key, end;     // tile number, its first key, end of its segment
    const char *k, *v;      // that key's vectors
};
// zeros into the chunks of `rows` tile rows that no fill writes
template <int NCH, int THREADS>
__device__ __forceinline__ void clear_tails(char* tile, int rows, int chunks) {
    if (chunks == NCH) return;
    for (int e = threadIdx.x; e < rows * NCH; e += THREADS) {
        const int r = e / NCH, c = (e % NCH) ^ swz<NCH>(r);
        if (c >= chunks) *(ix4*)(tile + e * 16) = ix4{0, 0, 0, 0};
    }
}
// Fill a [ROWS][NCH * 8] tile from any row addresses row(t) (null: zeros), zeros behind `chunks` 16-byte chunks.
template <int ROWS, int NCH, int NW, typename Row>
__device__ __forceinline__ void fill_rows(uint32_t tile, Row row_at, int chunks, int wave, int lane) {
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
__device__ __forceinline__ void fill_tile(uint32_t tile, const char* base, int64_t stride, int first, int end,
                                          int chunks, int wave, int lane) {
    fill_rows<ROWS, NCH, NW>(
        tile, [&](int t) { return first + t < end ? base + (int64_t)(first + t) * stride : nullptr; }, chunks, wave, lane);
}
// until at most N of this wave's loads are in flight: they finish in the order in which they were started
template <int N = 0>
__device__ __forceinline__ void wait_fills() {
    static_assert(N < 64, "the counter has 6 bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// loads that a wave issues for a [rows][nch * 8] tile: at least
constexpr int fill_loads(int rows, int nch, int nw) { return rows * nch / (nw * 64); }
// Tiles go round ST LDS buffers, ST - 1 of them in flight or in use.  Before tile t is read: until its own loads (NL a
// tile) are done, those of the up to ST - 2 tiles behind it still in flight; then a barrier, after which the buffer of tile
// t - 1 is free.
template <int ST, int NL>
__device__ __forceinline__ void wait_tile(int tiles_behind) {
    if (tiles_behind >= ST - 2) wait_fills<(ST - 2) * NL>();
    else wait_fills<0>();
    __syncthreads();
}
// 4 bytes per lane from memory to LDS, lane l's behind `to` + 4 l
__device__ __forceinline__ void load_lds4(const char* src, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(to)), "v"((uint64_t)(uintptr_t)src)
                 : "memory", "m0");
}

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

// Scores enter exp2 as z * (|scale| log2 e): the sign of the scale goes into the register operand, and a scale of 0
// becomes one too small to matter, so that a masked score of -inf stays one.
__device__ __forceinline__ float score_factor(float scale) { return fmaxf(fabsf(scale) * kLog2e, 1e-30f); }
__device__ __forceinline__ ix4 flip_sign(ix4 v, float scale) {
    const int s = scale < 0.f ? (int)0x80008000 : 0;
    return ix4{v.x ^ s, v.y ^ s, v.z ^ s, v.w ^ s};
}

// ---- Values that are not finite where nothing may be read from them ----
// A masked probability of 0 still lets an inf or NaN of its key's vector into the query's sums (0 * inf).  The
// kernels look at their sums at the end, and where one is not finite they run again carefully: operands enter
// the second product with their non-finite elements as 0, and those are added for the pairs that see them.
template <typename E>
__device__ __forceinline__ bool not_finite16(int half) {
    const int em = sizeof(E) == 2 && Half16<E>::kLift == 0.f ? 0x7f80 : 0x7c00;
    return (half & em) == em;
}
template <typename E>
__device__ __forceinline__ ix4 finite_part(ix4 v) {
    ix4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int lo = v[i] & 0xffff, hi = (v[i] >> 16) & 0xffff;
        o[i] = (not_finite16<E>(lo) ? 0 : lo) | ((not_finite16<E>(hi) ? 0 : hi) << 16);
    }
    return o;
}
// acc += the non-finite elements of operand a, for every pair that `see` (ones and zeros) marks
template <typename E>
__device__ __forceinline__ void add_not_finite(fx16& acc, ix4 a, ix4 see) {
    constexpr bool bf = Half16<E>::kLift == 0.f;
    const int em = bf ? 0x7f80 : 0x7c00, one = bf ? 0x3f80 : 0x3c00;
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) any |= not_finite16<E>(a[i] & 0xffff) || not_finite16<E>(a[i] >> 16 & 0xffff);
    if (!__any(any)) return;
#pragma unroll 1
    for (int c = 0; c < 3; ++c) {  // +inf, -inf, NaN
        ix4 ind;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int w = 0;
#pragma unroll
            for (int s = 0; s < 32; s += 16) {
                const int x = (a[i] >> s) & 0xffff;
                const bool is = c == 0 ? x == em : c == 1 ? x == (em | 0x8000) : (x & 0x7fff) > em;
                w |= (is ? one : 0) << s;
            }
            ind[i] = w;
        }
        fx16 n;
#pragma unroll
        for (int x = 0; x < 16; ++x) n[x] = 0.f;
        n = Half16<E>::mma(ind, see, n);
        const float v = c == 0 ? INFINITY : c == 1 ? -INFINITY : __builtin_nanf("");
#pragma unroll
        for (int x = 0; x < 16; ++x) acc[x] += n[x] > 0.f ? v : 0.f;
    }
}
template <typename E>
__device__ __forceinline__ int pack_ones(bool a, bool b) {
    constexpr int one = Half16<E>::kLift == 0.f ? 0x3f80 : 0x3c00;
    return (a ? one : 0) | (b ? one << 16 : 0);
}
// whether any of N registers holds a value that is not finite
template <int N>
__device__ __forceinline__ bool any_not_finite(const fx16 (&acc)[N], float with) {
    float t = with * 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
        for (int x = 0; x < 16; ++x) t = __builtin_fmaf(acc[c][x], 0.f, t);
    return !(t == 0.f);
}

// Writes a wave's 32 result rows of C 16-bit channels, 16 bytes a lane along the rows: from the registers directly
// every store would touch 32 rows.  acc: lane = row, registers = channels (times mul); tile: 32 * NCH * 16 bytes of
// LDS that are the wave's own; to(row): where the row goes, or null.
template <typename E, int NCH, int NA, typename Row>
__device__ __forceinline__ void store_rows(char* tile, const fx16 (&acc)[NA], float mul, int C, int lane, Row to) {
    const int h = lane >> 5, row = lane & 31;
#pragma unroll
    for (int c = 0; c < NA; ++c)
#pragma unroll
        for (int x = 0; x < 16; x += 4) {
            const int chunk = c * 4 + x / 4;  // channels c * 32 + 2 x + 4 h ..
            *(ix2*)(tile + (row * NCH + (chunk ^ swz<NCH>(row))) * 16 + h * 8) =
                ix2{pack2<E>(acc[c][x] * mul, acc[c][x + 1] * mul), pack2<E>(acc[c][x + 2] * mul, acc[c][x + 3] * mul)};
        }
    __builtin_amdgcn_wave_barrier();  // LDS keeps a wave's order; the compiler has to as well
    constexpr int PER = 64 / NCH > 0 ? 64 / NCH : 1;  // rows a load
    const int c = lane % NCH;
    if (c * 8 >= C) return;
#pragma unroll
    for (int n = 0; n < 32 / PER; ++n) {
        const int r = n * PER + lane / NCH;
        const ix4 v = *(const ix4*)(tile + (r * NCH + (c ^ swz<NCH>(r))) * 16);
        char* at = to(r);
        if (at) *(ix4*)(at + c * 16) = v;
    }
}

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace custma
