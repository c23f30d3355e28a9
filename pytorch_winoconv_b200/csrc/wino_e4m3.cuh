// Device helpers of the fully connected layers: activations and their slopes, and the 8-bit form of activations kept for the
// backward pass.
//
// Eight bits: 32 neighbours of the last dimension share a power of two 2^e, the smallest (from 2^-127 on) that brings the largest
// finite magnitude among them within e4m3's 448; each is x / 2^e rounded to e4m3 (half to even).  A power of two costs nothing of
// the four significant bits, and what comes back (q 2^e) has so few that bf16 and f16 hold it without another rounding: a product
// that reads it is the product of exactly what was kept.  Infinities and NaN come back as NaN.
#pragma once

#include "wino_sm100.cuh"

namespace wino {
namespace e4m3 {

constexpr int BLOCK = 32;

// Biased exponent of the scale of a block whose largest finite magnitude is `top` (f32 bit arithmetic: 448 = 1.75 * 2^8).
__device__ __forceinline__ uint32_t scale_byte(float top) {
  const uint32_t b = __float_as_uint(top);
  const int e = (int)(b >> 23) - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(e, 0);
}
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float scale_of(uint32_t byte) {      // 255 (not written by pack) is NaN
  return byte == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(byte == 0u ? 0x400000u : byte << 23);
}
__device__ __forceinline__ float finite_magnitude(float x) {
  const float a = fabsf(x);
  return a < __uint_as_float(0x7F800000u) ? a : 0.f;
}
// Two values as e4m3, the first in the low byte; of a block without infinities (NaN is NaN in any case).
__device__ __forceinline__ uint32_t pack2_finite(float a, float b, float inv) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b * inv), "f"(a * inv));
  return r;
}
// Two values as e4m3, the first in the low byte.
__device__ __forceinline__ uint32_t pack2(float a, float b, float inv) {
  const float inf = __uint_as_float(0x7F800000u), nan = __uint_as_float(0x7FC00000u);
  a = fabsf(a) < inf ? a * inv : nan;
  b = fabsf(b) < inf ? b * inv : nan;
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)v));
  return sm100::Pair16<__half>::unpack(h);
}
// The largest finite value of the type: a block's top may round up beyond it (65504 keeps as 65536).
template <typename T> __device__ __forceinline__ float largest();
template <> __device__ __forceinline__ float largest<__half>() { return 65504.f; }
template <> __device__ __forceinline__ float largest<__nv_bfloat16>() { return __uint_as_float(0x7F7F0000u); }
// Scales up to this biased exponent keep 448 times the scale within the type.
template <typename T> __device__ __forceinline__ uint32_t safe_byte() { return sizeof(T) == 2 && largest<T>() < 1e5f ? 127u + 7u : 127u + 119u; }
template <typename T> __device__ __forceinline__ float within(float v) {      // NaN passes
  const float m = largest<T>();
  return v > m ? m : v < -m ? -m : v;
}

}  // namespace e4m3

namespace act {

// The smooth activations are built from the hardware's 2^x and 1/x (each good to a few 2^-23 relative), far below the 2^-9 or
// 2^-12 that rounding a result to 16 bits costs: a kernel that passes over memory has about 30 instructions a value to spend.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float recip(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float LOG2E = 1.4426950408889634f;
// sqrt(2 / pi) and the cubic term of the tanh form of GELU; (1 + tanh u) / 2 = sigmoid(2 u)
constexpr float GELU_C = 0.7978845608028654f, GELU_A = 0.044715f;

__device__ __forceinline__ float sigmoid(float t) { return recip(1.f + exp2_fast(-LOG2E * t)); }
__device__ __forceinline__ float clamp16(float z) {      // NaN passes
  float y;
  asm("{\n\t.reg .f32 t;\n\tmin.NaN.f32 t, %1, 0f41800000;\n\tmax.NaN.f32 %0, t, 0fC1800000;\n\t}" : "=f"(y) : "f"(z));
  return y;
}
// sigmoid(2 u) of the tanh form; z within +-16, beyond which it is 0 or 1 in fp32.
__device__ __forceinline__ float gelu_sigmoid(float z, float z2) {
  return recip(1.f + exp2_fast(z * fmaf(z2, -2.f * LOG2E * GELU_C * GELU_A, -2.f * LOG2E * GELU_C)));
}
// The normal distribution's integral, and its density, with one exponential: erfc(x) = (a1 t + ... + a5 t^5) exp(-x^2) with
// t = 1 / (1 + p x) for x >= 0 (Abramowitz and Stegun, formula 7.1.26: within 1.5e-7 of erf).
__device__ __forceinline__ float normal(float z, float &density) {
  const float x = fabsf(z) * 0.7071067811865476f, e = exp2_fast(-LOG2E * x * x), t = recip(fmaf(0.3275911f, x, 1.f));
  const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
  const float tail = 0.5f * p * e;
  density = 0.3989422804014327f * e;
  return z < 0.f ? tail : 1.f - tail;
}

__device__ __forceinline__ float apply(float z, int act) {
  switch (act) {
    case WINOCONV_ACT_RELU: return z < 0.f ? 0.f : z;      // NaN passes
    case WINOCONV_ACT_GELU: { float d; return z * normal(z, d); }
    case WINOCONV_ACT_GELU_TANH: { const float c = clamp16(z); return z * gelu_sigmoid(c, c * c); }
    case WINOCONV_ACT_SILU: return z * sigmoid(z);
    default: return z;
  }
}
__device__ __forceinline__ float slope(float z, int act) {
  switch (act) {
    case WINOCONV_ACT_RELU: return z > 0.f ? 1.f : z <= 0.f ? 0.f : z;
    case WINOCONV_ACT_GELU: {
      float d;
      const float c = clamp16(z), n = normal(c, d);      // the density is 0 beyond
      return fmaf(c, d, n);
    }
    case WINOCONV_ACT_GELU_TANH: {
      const float c = clamp16(z), c2 = c * c, s = gelu_sigmoid(c, c2);
      return fmaf(c * fmaf(c2, 6.f * GELU_C * GELU_A, 2.f * GELU_C), fmaf(-s, s, s), s);
    }
    case WINOCONV_ACT_SILU: {
      const float s = sigmoid(z);
      return fmaf(z * s, 1.f - s, s);
    }
    default: return 1.f;
  }
}

}  // namespace act
}  // namespace wino
