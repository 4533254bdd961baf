// The 4-bit cache of keys and values: how a page is laid out, and what rounds to it.
//
// A kv head's values are held in groups of 32 dims.  A group keeps 32 codes of 4 bits and one scale s: a code c stands for
// (c - 8) * s with c - 8 in [-7, 7].  s is a seventh of the group's largest magnitude (the quotient in 32-bit) rounded to 5
// significant bits, so that every (c - 8) * s has at most 8 and is a bfloat16 number: unpacking rounds nothing, in any
// type, and a cache expanded to bfloat16 holds exactly what this one does.  The coarser scale costs at most 3 % of a step;
// a bfloat16 scale of all 8 bits would have made products of 11 bits, and every kernel with bfloat16 operands would have
// rounded them again.  A group whose largest magnitude is below 2^-100 holds zeros; a group with a number that is not
// finite reads back as NaN, all of it (its scale is NaN).
//
// 16 tokens of a kv head are one contiguous tile, the unit of every copy; a page of `page_size` tokens (a multiple of 16)
// is [kv head][page_size / 16] tiles.  A tile, for heads of hd = 32 G:
//     16 rows of hd / 2 bytes   codes of keys
//     16 rows of hd / 2 bytes   codes of values
//     16 rows of G bfloat16     scales of keys
//     16 rows of G bfloat16     scales of values
// Keys are the left operand of a product over dims and values that of a product over tokens, so the rows are ordered by
// who reads them (mma.m16n8k16; lane 4 e + t of a warp):
//     keys:    dim 32 g + 8 t + i is nibble i of 32-bit word t * G + g: lane t of a row takes its G words in one load
//     values:  dim 16 i + 2 e + j is nibble j of byte e * 2 G + i: lane e of a row takes its 2 G bytes in one load
#pragma once

#include "common.cuh"

#include <float.h>

constexpr int kKv4Tile = 16;                   // tokens of a tile
constexpr int kKv4Group = 32;                  // dims that share a scale

__host__ __device__ constexpr int kv4_tile_bytes(int hd) { return 18 * hd; }
__host__ __device__ constexpr int kv4_values_at(int hd) { return 8 * hd; }
__host__ __device__ constexpr int kv4_key_scales_at(int hd) { return 16 * hd; }
__host__ __device__ constexpr int kv4_value_scales_at(int hd) { return 17 * hd; }

// The scale of a group whose largest magnitude is `largest` (finite): 5 significant bits of the 32-bit quotient, ties to even.
__device__ __forceinline__ float kv4_scale(float largest) {
    if (largest < 7.888609052210118e-31f) return 0.f;          // 2^-100
    const uint32_t bits = __float_as_uint(__fdiv_rn(largest, 7.f));
    return __uint_as_float((bits + 0x3ffffu + (bits >> 19 & 1u)) & ~0x7ffffu);
}

// The whole number nearest to x / s, ties to even, plus 8; |x| is at most the group's largest magnitude (of which s is a seventh but
// for 1/32, so the number is from -7 to 7), and 0 where s is; `inverse` is about 1 / s.  The product in 32-bit may fall on the
// other side of a border between two numbers; what is left of x after k steps of s is exact in sign (k s has 8 bits), and settles it: a
// step more where it is above half of one, or is half and the number odd.  Adding 1.5 * 2^23 rounds to a whole number and leaves it in
// the low bits; magnitudes compare as their bits do.
__device__ __forceinline__ uint32_t kv4_code(float x, float s, float inverse) {
    constexpr float kWhole = 12582912.f;
    constexpr uint32_t kWholeBits = 0x4b400000u;
    const float t = fmaf(x, inverse, kWhole), left = fmaf(kWhole - t, s, x);
    uint32_t n = __float_as_uint(t);
    const uint32_t off = __float_as_uint(left) & 0x7fffffffu, half = __float_as_uint(0.5f * s);
    if (off + (n & 1u) > half) n += (uint32_t)(__float_as_int(left) >> 31 | 1);
    return n - (kWholeBits - 8u);
}
