// The 8-bit K/V cache: what its codes and exponent bytes mean, and the conversions to and from them.
//
// A token's row of one kv head (D values of K, or of V) is D codes in e4m3 and one exponent byte b:
//     value_d = code_d * 2^(b - 127)
// with e = b - 127 the smallest integer in [kMinExp, kMaxExp] for which every finite |x_d| <= 448 * 2^e (448: the
// largest code), and code_d = x_d * 2^-e rounded to nearest even. The scale is a power of two so that it rounds
// nothing: a code has at most four significant bits, so every value the cache stands for is a bf16 number, and the
// attention kernels may apply the scale to K, to the scores or to the probabilities with the same result. It costs
// no precision against an arbitrary scale either, because the codes are floating-point numbers themselves. Each row has its
// own: what is stored for a token depends on that token alone, not on what else was written to its block, in which
// order, or in how many calls.
//   inf and NaN become the NaN code; finite magnitudes above 448 * 2^kMaxExp saturate; an all-zero row takes kMinExp.
//   The range [-64, 63] keeps every product of a K or V value with the 2^+-64 of another row inside fp32 (not every product of
//   two such scales: the attention kernels multiply by one after the other).
#pragma once

#include <cuda_fp16.h>

#include "sbk_common.cuh"

namespace sbk {
namespace q8 {

constexpr int kMinExp = -64, kMaxExp = 63;

// exponent of a row whose largest finite magnitude is amax (>= 0, finite)
__device__ __forceinline__ int row_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  // amax = m * 2^k, m in [1, 2): it fits under 448 * 2^e = 1.75 * 2^(e + 8) with e = k - 8 when m <= 1.75
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < kMinExp ? kMinExp : (e > kMaxExp ? kMaxExp : e);   // (zero and subnormals have k = -127: kMinExp)
}
// 2^e for e in [-126, 127]
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// the scale of an exponent byte (the bytes this library writes lie in [63, 190]; any byte gives a finite scale)
__device__ __forceinline__ float byte_scale(uint32_t b) {
  return __uint_as_float(b == 255u ? 0x7f000000u : (b ? b << 23 : 0x00400000u));
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// two floats -> packed codes, `lo` in the low byte (nearest even, finite values saturate, NaN stays NaN)
__device__ __forceinline__ uint32_t pack_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// packed codes -> packed fp16 pair (exact)
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t w) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)w));
  return r;
}
// packed codes -> two floats (exact)
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t w) {
  const uint32_t h = e4m3x2_to_f16x2(w);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

}  // namespace q8
}  // namespace sbk
