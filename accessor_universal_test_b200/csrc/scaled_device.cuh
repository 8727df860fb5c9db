// scaled_device.cuh -- building blocks of the block-scaled 8-bit operators
// (sm_100a): element conversions and the encoding of a block.
#ifndef AUT_SCALED_DEVICE_CUH_
#define AUT_SCALED_DEVICE_CUH_

#include "autdot.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace aut::scaled {

constexpr int kBlock = 128; // columns (and, for weights, rows) of one scale

template <int Type> struct element;
template <> struct element<AUT_TYPE_FP32> { using type = float; };
template <> struct element<AUT_TYPE_BF16> { using type = __nv_bfloat16; };
template <> struct element<AUT_TYPE_FP16> { using type = __half; };
template <int Type> using element_t = typename element<Type>::type;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half narrow<__half>(float v) {
  return __float2half_rn(v);
}

// Largest code value F of a format.
template <int Code> __host__ __device__ constexpr float largest_code() {
  return Code == AUT_FP8_E4M3 ? 448.0f : 57344.0f;
}

// Two values to two codes (lo in the low byte): round to nearest even,
// magnitudes above F to F, NaN to the NaN code.
template <int Code> __device__ __forceinline__ uint32_t codes_of(float lo, float hi) {
  uint16_t r;
  if (Code == AUT_FP8_E4M3)
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// x / scale rounded to FP32, from the block's one reciprocal: Markstein's
// correction step (the residual x - q * scale is exact in one FMA) makes the
// product with the rounded reciprocal the correctly rounded quotient, so a
// value halfway between two codes goes the way of a true division; three
// operations a value where a division takes about ten.  (Below |x| = 2^-100
// the residual may underflow; the quotient is then within 2 ulp.)  An
// infinite x gives inf - inf = NaN, which encodes as NaN.
__device__ __forceinline__ float quotient(float x, float scale, float reciprocal) {
  const float q = x * reciprocal;
  return fmaf(fmaf(-q, scale, x), reciprocal, q);
}

// The scale of a block whose largest finite magnitude is `largest`: at least
// 2^-126, so that its reciprocal is finite and a block of zeros needs no case
// of its own.
template <int Code> __device__ __forceinline__ float scale_of(float largest) {
  constexpr float f = largest_code<Code>(), reciprocal = 1.0f / f;
  return fmaxf(quotient(largest, f, reciprocal), 1.17549435e-38f);
}

// |v| for a block's largest magnitude: infinities and NaN do not count.
__device__ __forceinline__ float finite_magnitude(float v) {
  const float a = fabsf(v);
  return a <= 3.40282347e38f ? a : 0.0f;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

} // namespace aut::scaled

#endif
