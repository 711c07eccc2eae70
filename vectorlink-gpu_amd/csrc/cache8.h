// The key/value cache in 8 bits: its layout, and what its kernels share beside cache.h.
//
// A page holds 64 tokens.  An element is a code of 8 bits (E4M3: sign, four bits of exponent, three of mantissa, no infinity, largest
// 448) times a power of two that a page's tokens share, one for the keys and one for the values of a head.  gfx950 turns two codes and
// such a power into two bfloat16 values in one instruction, and every value of the cache is exact in bfloat16: 4 significant bits,
// and the least power keeps the least code, 2^-9, a normal number.  A power of two means that a page whose power grows when a larger
// token comes (a page is written a token at a time) is rounded again only where codes become subnormal; a scale with a mantissa would
// round all 64 tokens anew at every growth.
//   keys    [pages, heads, 64, D]      a token's row is contiguous: 16 lanes x 4 read 16 tokens' rows in 16-byte pieces
//   values  [pages, heads, 16, D, 4]   a word is a dimension of 4 tokens, as the product with the weights sums over tokens
//   scales  [pages, heads]             a word: exponent + 127 of the keys, of the values, 1 where a token is not finite, 0
//   weights [pages, heads, 64]         accumulated weight of a token
//   positions [pages, heads, 64]       where it stood in its text
// A token with an element that is not finite is NaN codes all over.
#pragma once
#include "cache.h"

constexpr int kLeastExponent8 = -117;  // of a page's power: 2^-9 of it is 2^-126
constexpr int kMostExponent8 = 119;    // 448 of it is a float32; larger magnitudes become that
constexpr uint32_t kByteNaN = 127;     // without the sign

__device__ inline float power_of_byte(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }
// A page's powers.  Whatever a word holds - a page that was never written - they are powers that pages have.
__device__ inline uint32_t in_range(uint32_t byte) { return min(max(byte, (uint32_t)(kLeastExponent8 + 127)), (uint32_t)(kMostExponent8 + 127)); }
__device__ inline uint32_t byte_of_keys(uint32_t word) { return in_range(word & 255); }
__device__ inline uint32_t byte_of_values(uint32_t word) { return in_range(word >> 8 & 255); }
__device__ inline float scale_of_keys(uint32_t word) { return power_of_byte(byte_of_keys(word)); }
__device__ inline float scale_of_values(uint32_t word) { return power_of_byte(byte_of_values(word)); }
__device__ inline bool is_marked(uint32_t word) { return word >> 16 & 255; }

// two codes of the lower or upper half of a word as bfloat16
template <bool UPPER>
__device__ inline uint32_t two_of_bytes(uint32_t word, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, UPPER));
}
__device__ inline bf16x8 eight_of_bytes(uint32_t x, uint32_t y, float scale) {
    u32x4 v = {two_of_bytes<false>(x, scale), two_of_bytes<true>(x, scale), two_of_bytes<false>(y, scale), two_of_bytes<true>(y, scale)};
    return __builtin_bit_cast(bf16x8, v);
}
// the same as half precision; without the power every code is exact there
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
template <bool UPPER>
__device__ inline uint32_t two_halves(uint32_t word) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0f, UPPER));
}
__device__ inline f16x8 eight_halves(uint32_t x, uint32_t y) {
    u32x4 v = {two_halves<false>(x), two_halves<true>(x), two_halves<false>(y), two_halves<true>(y)};
    return __builtin_bit_cast(f16x8, v);
}
// What scores of such keys are multiplied with: the call's scale and the keys' power, kept a normal number - 0 would make NaN of scores
// that are masked, where the true product leaves all scores next to nothing all the same.  Where it leaves float32 it is the scale
// alone, and the scores take the power before (power_ahead): one of codes and half precision may be as little as 2^-33.
__device__ inline bool is_beyond(float scale, float power) { return scale * power > 0x1.fffffep127f; }
__device__ inline float scale_with(float scale, float power) { return is_beyond(scale, power) ? scale : fmaxf(scale * power, 0x1p-126f); }
__device__ inline float power_ahead(float scale, float power) { return is_beyond(scale, power) ? power : 1.0f; }
// the four codes of a word as numbers, and the way back: to the nearest code, of two as near the even one; magnitudes up to 448
__device__ inline f32x4 four_numbers(uint32_t word) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(word, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(word, true);
    return f32x4{a[0], a[1], b[0], b[1]};
}
__device__ inline uint32_t four_codes(f32x4 x) {
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], low, true);
}
__device__ inline f32x4 within(f32x4 x) {
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = __builtin_amdgcn_fmed3f(x[i], -448.0f, 448.0f);
    return x;
}
// 2^-n, for codes that are rounded to a power 2^n times as large: behind 2^-20 none is left
__device__ inline float power_below(uint32_t n) { return power_of_byte(127 - min(n, 64u)); }
// The byte of the least power whose 448-fold is not below a finite magnitude, given by its bits.
__device__ inline uint32_t fitting_byte(uint32_t bits) {
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFF) > 0x600000);  // 448 = 1.75 * 2^8
    return (uint32_t)(min(max(e, kLeastExponent8), kMostExponent8) + 127);
}

// ---- host side -------------------------------------------------------------
int vl_cache8_of(const vl_cache8 *cache, CacheView *out);
