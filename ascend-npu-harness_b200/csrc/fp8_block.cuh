// The 8-bit block format shared by the checkpointed operators and the 8-bit matrix product:
// e4m3 codes with one fp32 scale for each block of 128 elements of a row (activations,
// checkpoints) or for each 128 x 128 tile (weights).
//
//   amax  = max(max |x| over the block, 2^-100)
//   q     = e4m3(x * (448 / amax)), round to nearest even      448 = largest finite e4m3 value
//   scale = amax / 448,   x ~ q * scale
//
// Both quotients are correctly rounded fp32 divisions (one each per block), and the code is one
// fp32 product and one rounding, so any implementation of these three lines in fp32 gives the same
// bits.  The floor keeps 448 / amax finite for blocks that are zero or all subnormal.  The largest
// magnitude is taken as an integer maximum over the sign-less bit patterns, which orders finite
// values as numbers and lets an infinity or a NaN win: such a block gets scale inf or NaN and reads
// back as NaN everywhere, instead of hiding the fault in one element.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace hc {

constexpr uint32_t kFp8Block = 128;
constexpr float kFp8Max = 448.0f;
constexpr uint32_t kFp8FloorBits = 0x0D800000u;  // 2^-100

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// The block's amax from the bits of its largest magnitude.
__device__ __forceinline__ float fp8_amax(uint32_t bits) {
    return __uint_as_float(bits < kFp8FloorBits ? kFp8FloorBits : bits);
}
// Multiplier 448 / amax and scale amax / 448.
__device__ __forceinline__ void fp8_block_scale(uint32_t bits, float& inv, float& scale) {
    const float amax = fp8_amax(bits);
    inv = __fdiv_rn(kFp8Max, amax);
    scale = __fdiv_rn(amax, kFp8Max);
}

// Two values to two codes, a in the low byte.
__device__ __forceinline__ uint32_t fp8_encode2(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint8_t fp8_encode(float a) {
    return static_cast<uint8_t>(__nv_cvt_float_to_fp8(a, __NV_SATFINITE, __NV_E4M3));
}
// Two codes (low byte first) to two values; every e4m3 value is exact in half precision.
__device__ __forceinline__ float2 fp8_decode2(uint32_t two) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xFFFFu), __NV_E4M3);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ float fp8_decode(uint8_t one) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(one), __NV_E4M3);
    return __half2float(*reinterpret_cast<const __half*>(&h));
}

// max(|a|, |b|, |c|), NaN if any of them is.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
    float m;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}

__device__ __forceinline__ uint32_t warp_umax(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

}  // namespace hc
