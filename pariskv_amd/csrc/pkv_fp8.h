// Values in eight bits: e4m3 codes times a scale 2^e that a group of values shares, e the least whole number from -100 on with
// |x| <= 448 2^e for all finite x of the group (448 is the largest code).  e4m3 has the same relative precision whatever the scale, so a power
// of two costs nothing; dividing by it is exact, a code is rounded once, and a scale that grows leaves the codes of its group
// exact down to those that get below 2^-6.
#pragma once

#include "pkv_common.h"

#if defined(__HIPCC__)

constexpr int kFp8Least = -100;

// e for a largest magnitude given by its bits (0 for nothing; never an infinity).
__device__ __forceinline__ int fp8_exponent(uint32_t top) {
  const int e = (int)(top >> 23) - 135 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);  // 448 = 1.75 * 2^8
  return e < kFp8Least ? kFp8Least : e;
}
// 2^e, -126 <= e <= 127
__device__ __forceinline__ float fp8_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The bits of |x|, none for an infinity or a NaN.
__device__ __forceinline__ uint32_t fp8_magnitude(float x) {
  const uint32_t m = __float_as_uint(x) & 0x7fffffffu;
  return m < 0x7f800000u ? m : 0u;
}

// Two codes in the low half of a word, x * inv each: past 448 (infinities) 448, a NaN stays one.
__device__ __forceinline__ float fp8_limited(float x) { return x != x ? x : __builtin_amdgcn_fmed3f(x, -448.0f, 448.0f); }
__device__ __forceinline__ uint32_t fp8_codes4(float a, float b, float c, float d, float inv) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_limited(a * inv), fp8_limited(b * inv), 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_limited(c * inv), fp8_limited(d * inv), w, true);
  return (uint32_t)w;
}
__device__ __forceinline__ pkv_u32x2 fp8_codes8(const float (&x)[8], float inv) {
  return pkv_u32x2{fp8_codes4(x[0], x[1], x[2], x[3], inv), fp8_codes4(x[4], x[5], x[6], x[7], inv)};
}

// The four values of a word of codes.
__device__ __forceinline__ void fp8_values4(uint32_t w, float *x) {
  const pkv_f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
}
// ... of its lower (upper) half as two bf16 numbers, exact.
template <bool UPPER>
__device__ __forceinline__ uint32_t fp8_bf16x2(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, UPPER));
}

// Eight values of a row from 8 bf16 or fp32 numbers, 16-byte aligned.
template <bool BF16>
__device__ __forceinline__ void fp8_load8(const char *p, float (&x)[8]) {
  if constexpr (BF16) {
    const pkv_u32x4 w = *(const pkv_u32x4 *)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  } else {
    const float4 a = ((const float4 *)p)[0], b = ((const float4 *)p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
}

#endif
