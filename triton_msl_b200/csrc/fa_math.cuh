// Softmax arithmetic of the attention kernels: exponentials split between
// the MUFU and the FMA pipe, packed fp32 pairs, three-input maxima.
#pragma once
#include <cuda_runtime.h>

namespace b2 {
namespace fa {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- packed fp32x2 arithmetic (one issue slot for two lanes' worth of work)
typedef unsigned long long f2_t;
__device__ __forceinline__ f2_t f2_pack(float a, float b) {
  f2_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_unpack(f2_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ f2_t f2_fma(f2_t a, f2_t b, f2_t c) {
  f2_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2_t f2_mul(f2_t a, f2_t b) {
  f2_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2_t f2_add(f2_t a, f2_t b) {
  f2_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2_t f2_add_rm(f2_t a, f2_t b) {
  f2_t r;
  asm("add.rm.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x for two lanes on the FMA pipe, x <= 126; 0 from x = -127 down, so that a masked
// score (-inf) has no weight (2^-126 is a normal bf16, which a value of 1e38 brings back).
// Between -127 and -126 the result lies below 2^-126 and keeps no relative accuracy.
// Range reduction: t = x + 1.5*2^23 rounded toward -inf holds floor(x) in the
// low mantissa bits of t; f = x - floor(x) lies in [0, 1); 2^f comes from a
// cubic p(f) = 1 + f*(c1 + f*(c2 + f*c3)) whose coefficients are this file's
// own weighted least-squares fit of 2^f on [0, 1] with p(0) = 1 and p(1) = 2
// (max relative error 1.03e-4, below the fp16 / bf16 rounding of P); floor(x)
// is then added into the exponent field.
__device__ __forceinline__ void exp2_poly2(float x0, float x1, float& y0, float& y1) {
  constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23
  constexpr float c1 = 0.6954244f, c2 = 0.22630768f, c3 = 0.07826797f;
  // at -127: f = 0 and p = 1 exactly, whose bits less 127 << 23 are 0
  x0 = fmaxf(x0, -127.f);
  x1 = fmaxf(x1, -127.f);
  const f2_t x = f2_pack(x0, x1);
  const f2_t t = f2_add_rm(x, f2_pack(kMagic, kMagic));
  const f2_t xi = f2_add(t, f2_pack(-kMagic, -kMagic));
  const f2_t f = f2_fma(xi, f2_pack(-1.f, -1.f), x);
  f2_t p = f2_fma(f, f2_pack(c3, c3), f2_pack(c2, c2));
  p = f2_fma(f, p, f2_pack(c1, c1));
  p = f2_fma(f, p, f2_pack(1.f, 1.f));
  float p0, p1, t0, t1;
  f2_unpack(p, p0, p1);
  f2_unpack(t, t0, t1);
  // bits(t) << 23 == floor(x) << 23 (mod 2^32): the magic's own bits shift out.
  y0 = __int_as_float(__float_as_int(p0) + (__float_as_int(t0) << 23));
  y1 = __int_as_float(__float_as_int(p1) + (__float_as_int(t1) << 23));
}

}  // namespace fa
}  // namespace b2
