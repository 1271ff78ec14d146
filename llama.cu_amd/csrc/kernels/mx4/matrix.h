// The matrix instructions of the products with 4-bit weights: features are the rows of the result, tokens its columns.
#pragma once

// 16 features x 16 tokens of 32 k, and 32 x 32 of 16 k, bfloat16.
__device__ __forceinline__ mx4_f32x4 mx4_multiply_16(const mx4_u32x4 &features, const mx4_u32x4 &tokens, const mx4_f32x4 &sum) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mx4_bf16x8, features), __builtin_bit_cast(mx4_bf16x8, tokens), sum, 0, 0, 0);
}
__device__ __forceinline__ mx4_f32x16 mx4_multiply_32(const mx4_u32x4 &features, const mx4_u32x4 &tokens, const mx4_f32x16 &sum) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(mx4_bf16x8, features), __builtin_bit_cast(mx4_bf16x8, tokens), sum, 0, 0, 0);
}

// 16 x 16 of 128 k, and 32 x 32 of 64 k, codes of 4 bits: a lane has a block of 32 of its row, and its scale in byte BYTE of a register.
__device__ __forceinline__ mx4_i32x8 mx4_block(const mx4_u32x4 &codes) { return mx4_i32x8{(int)codes[0], (int)codes[1], (int)codes[2], (int)codes[3], 0, 0, 0, 0}; }
template <int BYTE>
__device__ __forceinline__ mx4_f32x4 mx4_multiply_codes_16(const mx4_u32x4 &features, const mx4_u32x4 &tokens, const mx4_f32x4 &sum, uint32_t feature_scales, uint32_t token_scales) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx4_block(features), mx4_block(tokens), sum, 4, 4, BYTE, (int)feature_scales, BYTE, (int)token_scales);
}
template <int BYTE>
__device__ __forceinline__ mx4_f32x16 mx4_multiply_codes_32(const mx4_u32x4 &features, const mx4_u32x4 &tokens, const mx4_f32x16 &sum, uint32_t feature_scales, uint32_t token_scales) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx4_block(features), mx4_block(tokens), sum, 4, 4, BYTE, (int)feature_scales, BYTE, (int)token_scales);
}
