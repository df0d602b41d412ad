// The 8-bit number format of the block-scaled projection and of the cache: an e4m3 code times a power of two. The
// exponent of a block whose largest finite magnitude is a is e = max(ceil(log2(a / 448)), -64), stored as the byte
// e + 127; codes are rounded to nearest even; what is not finite becomes NaN. A power of two costs no precision (the
// codes are floating point themselves), makes a change of scale exact down to the code's subnormals, and is what the
// block-scaled tensor-core instruction applies by itself.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace muse {

constexpr int FP8_E_MIN = -64;
constexpr int FP8_BLOCK = 128;   // columns (and weight rows) that share a scale in the projection

// |v| as the largest-magnitude search sees it: what is not finite does not count.
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.f;
}
// Exponent byte of a block: 448 = 1.75 * 2^8, so the exponent of a = f * 2^E (1 <= f < 2) is E - 8, or E - 7 when
// f > 1.75. FP32 subnormals lie far below the smallest exponent.
__device__ __forceinline__ int fp8_exponent_byte(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = static_cast<int>(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, FP8_E_MIN) + 127;
}
__device__ __forceinline__ float exp2_byte(int byte) { return __uint_as_float(static_cast<uint32_t>(byte) << 23); }   // 2^(byte - 127)
__device__ __forceinline__ float exp2_byte_inv(int byte) { return __uint_as_float(static_cast<uint32_t>(254 - byte) << 23); }

// Two values (already divided by the block's scale) to two codes, the first in the low byte. Round to nearest even;
// values beyond 448 saturate, infinities and NaN become NaN.
__device__ __forceinline__ uint32_t fp8_pack2(float lo, float hi) {
  lo = fabsf(lo) <= 3.402823466e38f ? lo : __uint_as_float(0x7fffffffu);
  hi = fabsf(hi) <= 3.402823466e38f ? hi : __uint_as_float(0x7fffffffu);
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) { return fp8_pack2(a, b) | fp8_pack2(c, d) << 16; }
// Codes of the low half of `v` (two bytes) as a pair of FP16 values: exact.
__device__ __forceinline__ uint32_t fp8_to_half2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}
__device__ __forceinline__ float2 fp8_to_float2(uint16_t v) {
  const uint32_t h = fp8_to_half2(v);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

}  // namespace muse
