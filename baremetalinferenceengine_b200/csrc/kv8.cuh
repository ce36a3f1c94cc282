// The 8-bit paged cache's numbers (bm_paged_kv8_t): e4m3 codes and, for each block of slots
// and head, a power of two that multiplies them.
//
// A power of two costs e4m3 nothing: its values are floating, so a scale below or above the
// best one by less than 2 only moves where they end (448) and where they thin out (2^-6).
// In return x 2^-E is exact, so a value is rounded once; a block whose scale grows has its
// earlier codes moved without a rounding, but for those that get below 2^-6; and attention
// adds exponents instead of multiplying.
#pragma once

#include <cuda_fp16.h>

#include "bm_common.cuh"
#include "bm_host.h"

namespace bm {
namespace kv8 {

// Exponents of a scale. 448 * 2^40 and 2^-49 are far outside what layers hold; within these
// bounds no product of two scales with a softmax weight that counts leaves fp32's range.
constexpr int kLowest = -40, kHighest = 40;

__device__ __forceinline__ float power(int e) { return __int_as_float((e + 127) << 23); }

// The exponent that a stored scale stands for (what the append never writes counts as the
// nearest that it does).
__device__ __forceinline__ int exponent(uint8_t scale) { return min(max(static_cast<int>(scale) - 127, kLowest), kHighest); }

// ceil(log2(amax / 448)) within the bounds: 448 = 1.75 * 2^8, so the mantissa decides.
__device__ __forceinline__ int exponent_for(uint32_t amax_bits) {
  const int e = static_cast<int>(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kLowest), kHighest);
}

// |x| as bits, which order as the values do, from kNotFinite on the infinities and NaN.
constexpr uint32_t kNotFinite = 0x7f800000u;
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Two values to two codes (lo in the low byte): nearest even, ends at +-448, NaN stays one. (An infinity would end at
// 448, too: it is made NaN before.)
__device__ __forceinline__ uint32_t to_codes(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Four codes of a word as four values.
__device__ __forceinline__ void from_codes(uint32_t w, float* f) {
  uint32_t a, b;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(a) : "h"(static_cast<uint16_t>(w)));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b) : "h"(static_cast<uint16_t>(w >> 16)));
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
  f[0] = x.x;
  f[1] = x.y;
  f[2] = y.x;
  f[3] = y.y;
}

}  // namespace kv8

// Host checks of an 8-bit paged cache's description, shared by its entry points.
int check_paged_kv8(const char* what, const bm_paged_kv8_t* cache);
// Whether `bytes` from p on share memory with a checked cache's pages or scales.
bool meets_pages8(const bm_paged_kv8_t& cache, const void* p, uintptr_t bytes);

}  // namespace bm
