// What the kernels of the 8-bit paged cache share.
//
// Cache layout: key / value codes [num_layers, num_blocks, block_size,
// kv_heads, head_dim] in e4m3, contiguous, and one fp32 scale per layer,
// block and kv head, [num_layers, num_blocks, kv_heads]: the value of a code
// is code * scale.  The appending kernels write powers of two in
// [2^-48, 2^48]; the readers take any finite positive scale of that range.
#pragma once

#include <cuda_fp8.h>

#include "nie_common.cuh"

namespace nie {

constexpr float kE4m3Max = 448.f;
constexpr float kScaleMin = 3.5527136788005009e-15f;  // 2^-48
constexpr float kScaleMax = 281474976710656.f;        // 2^48

// Two e4m3 codes (low byte first) as an f16 pair, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t c) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}

// Two floats as e4m3 codes, `lo` in the low byte; round to nearest even,
// magnitudes above 448 give 448, NaN gives NaN.
__device__ __forceinline__ uint16_t floats_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float e4m3_to_float(uint8_t c) {
  const uint32_t h = e4m3x2_to_f16x2((uint16_t)c);
  return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}

__device__ __forceinline__ float2 f16x2_to_float2(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

}  // namespace nie
