// The key/value cache in 4 bits: its layout, and what its kernels share.
//
// A page holds 64 tokens.  32 dimensions of a token are a group: 32 codes (E2M1: sign, two bits of exponent, one of mantissa) and
// one byte, the exponent + 127 of the power of two that the codes are multiplied with (the block format MXFP4 of the OCP
// microscaling specification).  gfx950 turns a byte of two codes and such an exponent into two bfloat16 values in one
// instruction, and every value of the cache is exact in bfloat16: 2 significant bits, exponents from -125 to 127.
//   keys    [pages, heads, 64, D / 2]          a token's row is contiguous: 16 lanes x 4 read 16 tokens' rows in 16-byte pieces
//   values  [pages, heads, 16, D / 8, 4, 4]    8 dimensions of 4 tokens are 16 bytes: the product with the weights sums over
//                                              tokens, so a lane needs several tokens of few dimensions
//   scales  [pages, heads, D / 32, 64]         the bytes of 4 tokens are a word
//   bounds  [pages, heads, 2, D]               largest and smallest key of the page in each dimension, 8 bits
//   bound_scales [pages, heads]                their power of two; kBoundless where a key or value is not finite
#pragma once
#include <type_traits>

#include "vl_common.h"

constexpr int kPage = 64;             // tokens
constexpr int kLeastExponent = -124;  // of a group's scale: half of it is still a normal bfloat16
constexpr int kNotFinite = 255;       // a scale's byte: the token held an infinity or a NaN, and reads as NaN
constexpr int kBoundless = 127;       // a page's bound_scale: no bounds

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct CacheView {
    int64_t pages;
    int heads, dim;
    uint8_t *keys, *key_scales, *values, *value_scales;
    int8_t *bounds, *bound_scales;
    // of a cache in 8 bits (cache8.h), which has none of the scales and bounds above
    uint32_t *scales;
    float *weights;
    int32_t *positions;
};

// The tokens of a call: rows [offsets[b], offsets[b + 1]) are new tokens of sequence b (offsets == nullptr: row b alone), whose
// blocks of 64 tokens lie on the pages table[b, :].
struct Tokens {
    const int32_t *table, *lengths, *offsets;
    int64_t table_stride;
    int rows, sequences, blocks;
};

// Rows of a sequence.  What the caller's offsets say is cut to the rows that there are, whatever they hold.
__device__ inline int first_row(const Tokens &t, int b) {
    if (!t.offsets) return b;
    return min(max(t.offsets[b], 0), t.rows);
}
__device__ inline int row_count(const Tokens &t, int b) {
    if (!t.offsets) return 1;
    return max(first_row(t, b + 1) - first_row(t, b), 0);
}
// The sequence of a row: the last whose first row is not behind it.
__device__ inline int sequence_of(const Tokens &t, int row) {
    if (!t.offsets) return row;
    int lo = 0, hi = t.sequences - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.offsets[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
// Whether a row is one of that sequence's: rows before the first offset and behind the last are nobody's.
__device__ inline bool is_row_of(const Tokens &t, int b, int row) {
    return row >= first_row(t, b) && row - first_row(t, b) < row_count(t, b);
}
// Length of a sequence, cut to what its table can name.
__device__ inline int length_of(const Tokens &t, int b) {
    return (int)min((int64_t)max(t.lengths[b], 0), (int64_t)t.blocks * kPage);
}
// The page of a block, or -1.
__device__ inline int64_t page_of(const Tokens &t, const CacheView &c, int b, int block) {
    if (block < 0 || block >= t.blocks) return -1;
    const int64_t p = t.table[b * t.table_stride + block];
    return p >= 0 && p < c.pages ? p : -1;
}

struct Piece {
    int sequence, piece;
};
// Which piece of which sequence is the w-th of all, where sequence b has pieces(b) of them; {-1, 0} behind the last.  All
// lanes of a wavefront take part and get the same answer.
template <class F>
__device__ inline Piece find_piece(int sequences, int w, F pieces) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < sequences; base += kWave) {
        const int n = base + lane < sequences ? pieces(base + lane) : 0;
        int sum = n;
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const int other = __shfl_up(sum, d);
            if (lane >= d) sum += other;
        }
        const int all = __shfl(sum, kWave - 1);
        if (w < before + all) {
            const int at = __ffsll((unsigned long long)__ballot(w < before + sum)) - 1;
            return {__builtin_amdgcn_readfirstlane(base + at),
                    __builtin_amdgcn_readfirstlane(w - before - __shfl(sum - n, at))};
        }
        before += all;
    }
    return {-1, 0};
}

// The types of queries, keys, values and outputs, by how many bfloat16 values hold one exactly.
template <int NS> struct ElementOf;
template <> struct ElementOf<1> { typedef __bf16 type; };
template <> struct ElementOf<2> { typedef _Float16 type; };
template <> struct ElementOf<3> { typedef float type; };

// 8 elements that lie on a boundary of their own type: gfx950 loads 16 bytes from any address, so there is no other path for rows
// off 16-byte boundaries.
template <int NS>
using Eight = typename ElementOf<NS>::type __attribute__((ext_vector_type(8)));
template <int NS>
__device__ inline Eight<NS> load8(const typename ElementOf<NS>::type *p) {
    typedef Eight<NS> Anywhere __attribute__((aligned(sizeof(typename ElementOf<NS>::type))));
    return *reinterpret_cast<const Anywhere *>(p);
}
// The same where `real`, else zeros; p is readable all the same.  A load behind a branch would be waited for before the next.
template <int NS>
__device__ inline Eight<NS> load8(const typename ElementOf<NS>::type *p, bool real) {
    typedef typename ElementOf<NS>::type E;
    Eight<NS> v = load8<NS>(p);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = real ? v[i] : (E)0.0f;
    return v;
}
template <int NS>
__device__ inline void store8(typename ElementOf<NS>::type *p, const float (&x)[8]) {
    typedef typename ElementOf<NS>::type E;
    typedef E e8 __attribute__((ext_vector_type(8)));
    e8 v;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (E)x[i];
    *reinterpret_cast<e8 *>(p) = v;
}

// A scale's byte `at` of a word as the operand of the conversions, which look at bits 23 to 30 alone.
__device__ inline float scale_at(uint32_t word, int at) {
    return __builtin_bit_cast(float, __builtin_amdgcn_alignbit(word, word, (8 * at + 9) & 31));
}
// two codes of byte B of a word as bfloat16
template <int B>
__device__ inline uint32_t two_values(uint32_t word, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, B));
}
__device__ inline bf16x8 eight_values(uint32_t word, float scale) {
    u32x4 v = {two_values<0>(word, scale), two_values<1>(word, scale), two_values<2>(word, scale), two_values<3>(word, scale)};
    return __builtin_bit_cast(bf16x8, v);
}
// f over the lanes l, l ^ 16, l ^ 32, l ^ 48
template <class F>
__device__ inline float over_quads(float x, F f) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t a0 = a[0], a1 = a[1];  // bit_cast of a vector's element takes the first one
    const uint32_t v = __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const uint32_t b0 = b[0], b1 = b[1];
    return f(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}
__device__ inline float max_over_quads(float x) {
    return over_quads(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ inline float sum_over_quads(float x) {
    return over_quads(x, [](float a, float b) { return a + b; });
}

// ---- host side -------------------------------------------------------------
// Checks what every entry point with a cache and a batch of tokens takes, and fills the kernels' structs; VL_OK or an error.
int vl_cache_of(const vl_cache *cache, CacheView *out);
int vl_tokens_of(const vl_tokens *tokens, Tokens *out);

// Sequences that have a row, at most: each may end inside a tile of its own
static inline int64_t sequences_with_rows(const Tokens &t) { return t.rows < t.sequences ? t.rows : t.sequences; }

// f(std::integral_constant<int, dim>) for a cache's row length
template <class F>
static inline void for_dim(int dim, F f) {
    switch (dim) {
        case 32: return f(std::integral_constant<int, 32>());
        case 64: return f(std::integral_constant<int, 64>());
        case 96: return f(std::integral_constant<int, 96>());
        case 128: return f(std::integral_constant<int, 128>());
        case 192: return f(std::integral_constant<int, 192>());
        case 256: return f(std::integral_constant<int, 256>());
    }
}
