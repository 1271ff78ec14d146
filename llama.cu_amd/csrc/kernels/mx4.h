// Microscaled 4-bit numbers: 32 neighbours along k share a power of two 2^(e - 127), held as the byte e (255: not a number, and with it
// all 32); a number is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (two bits of exponent, one of mantissa), two codes a byte, the first
// in the low half.
//
// A weight that is multiplied lies in the products' order: k filled up with zeros to pairs of 128, features to tiles of 16, and for every
// tile and pair of macro-steps (256 k)
//   codes   2 KB: [macro-step][group g = 0 .. 3][row of the tile] 16 bytes, the block of 32 that begins at k = 128 macro + 32 g: a wave's
//           load of 16 bytes a lane is one run of 1 KB and is an operand of the matrix instructions as it arrives;
//   scales  128 bytes: [row][odd][slice], a row's eight blocks together, block 2 slice + odd: the lane of a product of 32 x 32 x 64 that has the row's even or odd blocks finds its
//           four side by side.
#pragma once
#include "common.h"

typedef __attribute__((ext_vector_type(2))) __bf16 mx4_bf16x2;
typedef __attribute__((ext_vector_type(8))) __bf16 mx4_bf16x8;
typedef __attribute__((ext_vector_type(2))) float mx4_f32x2;
typedef __attribute__((ext_vector_type(4))) float mx4_f32x4;
typedef __attribute__((ext_vector_type(16))) float mx4_f32x16;
typedef __attribute__((ext_vector_type(4))) uint32_t mx4_u32x4;
typedef __attribute__((ext_vector_type(8))) int mx4_i32x8;

constexpr int MX4_BLOCK = 32, MX4_PAIR = 256;     // k that share a scale; k of a pair of macro-steps
constexpr int MX4_PAIR_CODES = 2048, MX4_PAIR_SCALES = 128;     // bytes of a tile of 16 features

// The scale's byte as the conversions take it: the exponent field of a float (they read 0 as 2^-127 and 255 as not a number).
__device__ __forceinline__ float mx4_scale(uint32_t e) { return __uint_as_float(e << 23); }

// Eight codes as bfloat16, scaled: exact, but for what lies beyond bfloat16's range.
__device__ __forceinline__ mx4_u32x4 mx4_to_bf16(uint32_t codes, float scale) {
    mx4_u32x4 v;
    v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
    v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
    v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
    v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
    return v;
}

// Where the scale of block b (0 .. 7) of a row's pair stands.
__device__ __forceinline__ int mx4_scale_place(int b) { return (b & 1) * 4 + (b >> 1); }

// Where row `row` of a weight in the products' order begins in its tile's first pair: bytes.
__device__ __forceinline__ size_t mx4_row_codes(int row, int pairs) { return (size_t)(row >> 4) * pairs * MX4_PAIR_CODES + (row & 15) * 16; }
__device__ __forceinline__ size_t mx4_row_scales(int row, int pairs) { return (size_t)(row >> 4) * pairs * MX4_PAIR_SCALES + (row & 15) * 8; }
