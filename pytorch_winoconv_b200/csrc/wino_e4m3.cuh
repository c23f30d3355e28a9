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
template <typename T> __device__ __forceinline__ float within(float v) {      // NaN passes
  const float m = largest<T>();
  return v > m ? m : v < -m ? -m : v;
}

}  // namespace e4m3

namespace act {

// sqrt(2 / pi) and the cubic term of the tanh form of GELU
constexpr float GELU_C = 0.7978845608028654f, GELU_A = 0.044715f;

// 1 / (1 + exp(-t)): with the hardware's exponential and division (a few 2^-23 relative), far below the 2^-9 or 2^-12 that
// rounding the result to 16 bits costs.
__device__ __forceinline__ float sigmoid(float t) { return __fdividef(1.f, 1.f + __expf(-t)); }

__device__ __forceinline__ float apply(float z, int act) {
  switch (act) {
    case WINOCONV_ACT_RELU: return z < 0.f ? 0.f : z;      // NaN passes
    case WINOCONV_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.7071067811865476f));
    case WINOCONV_ACT_GELU_TANH: return z * sigmoid(2.f * GELU_C * (z + GELU_A * z * z * z));      // (1 + tanh u) / 2 = sigmoid(2 u)
    case WINOCONV_ACT_SILU: return z * sigmoid(z);
    default: return z;
  }
}
__device__ __forceinline__ float slope(float z, int act) {
  switch (act) {
    case WINOCONV_ACT_RELU: return z > 0.f ? 1.f : z <= 0.f ? 0.f : z;
    case WINOCONV_ACT_GELU: return 0.5f * (1.f + erff(z * 0.7071067811865476f)) + z * __expf(-0.5f * z * z) * 0.3989422804014327f;
    case WINOCONV_ACT_GELU_TANH: {
      const float s = sigmoid(2.f * GELU_C * (z + GELU_A * z * z * z)), c = fminf(fmaxf(z, -16.f), 16.f);      // s (1 - s) is 0 beyond
      return s + c * s * (1.f - s) * (2.f * GELU_C) * (1.f + 3.f * GELU_A * c * c);
    }
    case WINOCONV_ACT_SILU: {
      const float s = sigmoid(z);
      return s * (1.f + z * (1.f - s));
    }
    default: return 1.f;
  }
}

}  // namespace act
}  // namespace wino
