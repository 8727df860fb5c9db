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

// Two FP32 values in one register pair: one instruction for both.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

// The scale of a block and its reciprocal as the sum of two FP32 values.
struct block_scale {
  float scale, inverse, rest;
};

// From the block's largest finite magnitude.  The scale, largest / F rounded
// once, is at least 2^-126: its reciprocal is then finite and a block of zeros
// needs no case of its own.  The division by the constant F is a product with
// 1 / F and Markstein's correction (the residual is exact in one FMA).  The
// reciprocal starts from the hardware's approximation r, within an ulp; with
// e = 1 - scale r, one FMA, 1 / scale = r + r (e + e^2) up to r e^3.  So rounded,
// inverse is 1 / scale rounded down (checked with all 2^23 fractions of a scale
// and every r within an ulp of the nearest value), and what is left of it is made
// the same way, now with an exact e.
template <int Code> __device__ __forceinline__ block_scale scale_of(float largest) {
  constexpr float f = largest_code<Code>(), reciprocal = 1.0f / f;
  block_scale s;
  const float q = largest * reciprocal;
  s.scale = fmaxf(fmaf(fmaf(-q, f, largest), reciprocal, q), 1.17549435e-38f);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s.scale));
  float e = fmaf(-s.scale, r, 1.0f);
  s.inverse = __fmaf_rd(r, __fmaf_ru(e, e, e), r);
  e = fmaf(-s.scale, s.inverse, 1.0f);
  s.rest = __fmul_rz(s.inverse, __fmaf_ru(e, e, e));
  return s;
}

// x / scale for two values, finite or NaN.  x * inverse + x * rest is within
// 2^-45 of the quotient before its one rounding to FP32.  Codes are those of a
// quotient rounded once: a tie between codes is met exactly, and where FP32 rounds
// to a tie what is beside it, the quotient lies at least 2^-49 from the midpoint
// that decides; all 712 pairs of fractions of scale and value that lie within 2^-43 of
// one were checked and come out right (with the roundings of scale_of, not with
// others).  The rest is not negative, so a zero keeps its sign.  Two operations for
// two values, where a division takes about ten for each.  Scales are at most
// kLargeScale here: the rest of a larger one's inverse would lose digits below the
// normal range.
__device__ __forceinline__ float2 quotient(float2 x, const block_scale &s) {
  return fma2(x, make_float2(s.inverse, s.inverse), mul2(x, make_float2(s.rest, s.rest)));
}

// Blocks with larger values are encoded times kDown, their scale times kUp.  What that
// takes below the normal range has a quotient that rounds to zero.
constexpr float kLargeScale = 0x1p100f, kDown = 0x1p-64f, kUp = 0x1p64f;

// |v| for a block's largest magnitude: infinities and NaN do not count.
__device__ __forceinline__ float finite_magnitude(float v) {
  const float a = fabsf(v);
  return a <= 3.40282347e38f ? a : 0.0f;
}

// Largest over the warp of values that are not negative, NaN passed over: their
// bit patterns order as integers.
__device__ __forceinline__ float warp_max(float v) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(v, 0.0f))));
}

// The same over each half of the warp: two reductions of the whole warp, since
// a reduction under two masks would part the halves' ways.
__device__ __forceinline__ float half_warp_max(float v, int lane) {
  const float low = warp_max(lane < 16 ? v : 0.0f), high = warp_max(lane < 16 ? 0.0f : v);
  return lane < 16 ? low : high;
}

} // namespace aut::scaled

#endif
