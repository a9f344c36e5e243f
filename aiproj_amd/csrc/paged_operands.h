// Operands of the paged-attention kernels on the gfx950 matrix cores: widening of e4m3fn codes, the
// products, wave-uniform values, and where a 16-token tile of a paged cache lies.
#pragma once

#include "kvfp8_common.h"

#include <type_traits>

namespace kvfp8 {

namespace {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ int32_t uniform(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ __forceinline__ int64_t uniform64(int64_t x) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int32_t)(uint32_t)x);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int32_t)(uint32_t)((uint64_t)x >> 32));
    return (int64_t)(((uint64_t)hi << 32) | lo);
}

__device__ __forceinline__ bf16x8_t cat8(bf16x2_t a, bf16x2_t b, bf16x2_t c, bf16x2_t d) {
    const bf16x4_t ab = __builtin_shufflevector(a, b, 0, 1, 2, 3);
    const bf16x4_t cd = __builtin_shufflevector(c, d, 0, 1, 2, 3);
    return __builtin_shufflevector(ab, cd, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Two e4m3fn codes (bytes 0-1 or 2-3 of x) -> two bf16, exact.
__device__ __forceinline__ bf16x2_t fp8x2_lo(uint32_t x) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false);
}
__device__ __forceinline__ bf16x2_t fp8x2_hi(uint32_t x) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true);
}

// Eight codes (x0 bytes 0..3, then x1) -> bf16x8 in byte order.
__device__ __forceinline__ bf16x8_t fp8x8(uint32_t x0, uint32_t x1) {
    return cat8(fp8x2_lo(x0), fp8x2_hi(x0), fp8x2_lo(x1), fp8x2_hi(x1));
}

__device__ __forceinline__ f32x4_t mma(bf16x8_t a, bf16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mma(f16x8_t a, f16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Operand type of the products: bf16 (e4m3fn codes widen to it exactly, bf16 caches
// are it), or f16 for an f16 cache read with f16 q (both exact in f16).
template <bool kF16> using OpT = std::conditional_t<kF16, f16x8_t, bf16x8_t>;
template <bool kF16> using OpE = std::conditional_t<kF16, _Float16, __bf16>;

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Global row (page * block_size + token base) of a 16-token tile; 0 when the
// page entry is outside the pool (the tile's tokens are then masked).
struct TileRef {
    int64_t row0;
    int32_t valid;
};

typedef const __attribute__((address_space(4))) int32_t* const_i32_ptr;

}  // namespace

}  // namespace kvfp8
