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

// The smooth activations are built from the hardware's 2^x and 1/x (each good to a few 2^-23 relative) and keep a relative error of
// 2^-18 plus what the argument of the exponential loses (2^-23 of its size, which is below 16 for results that f16 holds and below 128
// for bf16's; results below 2^-126 are 0): far below the 2^-9 or 2^-12 that rounding a result to 16 bits costs.  They work on two values
// an instruction: a kernel that passes over memory at 6.5 TB/s has about 20 instructions a value to spend.
struct F2 {      // two fp32 values
  uint64_t v;
  F2() = default;
  __device__ __forceinline__ F2(uint64_t x) : v(x) {}
  __device__ __forceinline__ F2(float a, float b) : v(f2_pack(a, b)) {}
  __device__ __forceinline__ F2(float a) : v(f2_pack(a, a)) {}
  __device__ __forceinline__ float lo() const { float a, b; f2_unpack(v, a, b); return a; }
  __device__ __forceinline__ float hi() const { float a, b; f2_unpack(v, a, b); return b; }
};
__device__ __forceinline__ F2 operator+(F2 a, F2 b) { return F2(f2_add(a.v, b.v)); }
__device__ __forceinline__ F2 operator*(F2 a, F2 b) { return F2(f2_mul(a.v, b.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { return F2(f2_fma(a.v, b.v, c.v)); }
template <typename Op> __device__ __forceinline__ F2 each(F2 a, Op op) { return F2(op(a.lo()), op(a.hi())); }

__device__ __forceinline__ F2 exp2_fast(F2 x) {
  return each(x, [](float t) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t)); return y; });
}
__device__ __forceinline__ F2 recip(F2 x) {
  return each(x, [](float t) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t)); return y; });
}
constexpr float LOG2E = 1.4426950408889634f;
// sqrt(2 / pi) and the cubic term of the tanh form of GELU; (1 + tanh u) / 2 = sigmoid(2 u)
constexpr float GELU_C = 0.7978845608028654f, GELU_A = 0.044715f;

__device__ __forceinline__ F2 sigmoid(F2 t) { return recip(exp2_fast(t * F2(-LOG2E)) + F2(1.f)); }
// sigmoid(2 u) of the tanh form.  z2: z squared, at most 256: sigmoid is 0 or 1 in fp32 from |z| = 16 on, and nothing overflows.
__device__ __forceinline__ F2 square256(F2 z) { return each(z * z, [](float t) { return fminf(t, 256.f); }); }
__device__ __forceinline__ F2 gelu_sigmoid(F2 z, F2 z2) {
  return recip(exp2_fast(z * fma2(z2, F2(-2.f * LOG2E * GELU_C * GELU_A), F2(-2.f * LOG2E * GELU_C))) + F2(1.f));
}
// The normal distribution's integral, and its density, with one exponential.  For x >= 0 the integral from x on is exp(-x^2 / 2) g(x),
// where g falls from 1/2 like 1 / (x sqrt(2 pi)): here a polynomial in t = 1 / (1 + p x) without a constant term, p and its
// coefficients fitted (linear program on 2700 points of 0..13.5) for the smallest relative error, 5.3e-7; 1.5e-6 with fp32 steps up to
// x = 8, 4e-6 up to 13.2, where the exponential ends.  The relative error is what counts: GELU of a far negative z is z times the tail
// (a tail that is good to 1e-7 absolutely is off by 5e-4 of its value at -4 and 4e-3 at -6).
__device__ __forceinline__ F2 normal(F2 z, F2 &density) {
  const F2 x = each(z, [](float t) { return fabsf(t); });
  const F2 e = exp2_fast(z * z * F2(-0.5f * LOG2E)), t = recip(fma2(x, F2(0.26389465f), F2(1.f)));
  F2 p = fma2(t, F2(-0.06941466f), F2(0.20421680f));
  p = fma2(t, p, F2(-0.07724253f));
  p = fma2(t, p, F2(0.14928270f));
  p = fma2(t, p, F2(0.08021010f));
  p = fma2(t, p, F2(0.10781857f));
  p = fma2(t, p, F2(0.10512876f));
  const F2 tail = p * t * e, body = fma2(tail, F2(-1.f), F2(1.f));
  density = e * F2(0.3989422804014327f);
  return F2(z.lo() < 0.f ? tail.lo() : body.lo(), z.hi() < 0.f ? tail.hi() : body.hi());
}

__device__ __forceinline__ F2 apply(F2 z, int act) {
  switch (act) {
    case WINOCONV_ACT_RELU: return each(z, [](float t) { return t < 0.f ? 0.f : t; });      // NaN passes
    case WINOCONV_ACT_GELU: { F2 d(0.f); return z * normal(z, d); }
    case WINOCONV_ACT_GELU_TANH: return z * gelu_sigmoid(z, square256(z));
    case WINOCONV_ACT_SILU: return z * sigmoid(z);
    default: return z;
  }
}
// (products that could be 0 x infinity for large z are taken in the order that keeps them 0)
__device__ __forceinline__ F2 slope(F2 z, int act) {
  switch (act) {
    case WINOCONV_ACT_RELU: return each(z, [](float t) { return t > 0.f ? 1.f : t <= 0.f ? 0.f : t; });
    case WINOCONV_ACT_GELU: {
      F2 d(0.f);
      const F2 n = normal(z, d);
      return fma2(z, d, n);
    }
    case WINOCONV_ACT_GELU_TANH: {
      const F2 z2 = square256(z), s = gelu_sigmoid(z, z2);
      const F2 h = fma2(s * F2(-1.f), s, s) * z;
      return fma2(h, fma2(z2, F2(6.f * GELU_C * GELU_A), F2(2.f * GELU_C)), s);
    }
    case WINOCONV_ACT_SILU: {
      const F2 s = sigmoid(z);
      return fma2(z * s, fma2(s, F2(-1.f), F2(1.f)), s);
    }
    default: return F2(1.f);
  }
}

}  // namespace act
}  // namespace wino
