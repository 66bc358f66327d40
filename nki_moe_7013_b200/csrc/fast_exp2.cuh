// exp2 on the FMA pipe, two values at a time, and the packed fp32 arithmetic
// of sm_100 that it is built from.
//
// The special-function unit gives 16 results a cycle and SM; a softmax that
// feeds the tensor cores needs more.  2^x = 2^n 2^f with n the integer nearest
// to x and f = x - n in [-1/2, 1/2]: n comes from adding 1.5 * 2^23 (the sum's
// low mantissa bits are n), 2^f from a polynomial, 2^n from n shifted into an
// exponent.  The polynomial is the degree-5 minimax one of the relative error
// on [-1/2, 1/2], found by Remez exchange: 7.5e-8, 2.1e-7 with its fp32
// roundings -- as good as the unit's.  A NaN stays NaN; x below -126 gives
// 2^-126.
#pragma once

#include <stdint.h>

namespace qmoe {

typedef unsigned long long f32x2;  // two fp32, the lower one in the low half

__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x of both halves as p (the polynomial) and s (the power of two): 2^x = p * s.
__device__ __forceinline__ void exp2_poly2(f32x2 x, f32x2& p, f32x2& s) {
  float lo, hi;
  unpack2(x, lo, hi);
  const f32x2 xc = pack2(max_nan(lo, -126.f), max_nan(hi, -126.f));
  const f32x2 t = add2(xc, pack2(12582912.f, 12582912.f));
  const f32x2 f = add2(xc, fma2(t, pack2(-1.f, -1.f), pack2(12582912.f, 12582912.f)));
  p = pack2(0.0013276472454890609f, 0.0013276472454890609f);
  p = fma2(p, f, pack2(0.009675540961325169f, 0.009675540961325169f));
  p = fma2(p, f, pack2(0.05550713092088699f, 0.05550713092088699f));
  p = fma2(p, f, pack2(0.24022120237350464f, 0.24022120237350464f));
  p = fma2(p, f, pack2(0.6931469440460205f, 0.6931469440460205f));
  p = fma2(p, f, pack2(1.0000001192092896f, 1.0000001192092896f));
  float tl, th;
  unpack2(t, tl, th);
  s = pack2(__uint_as_float((__float_as_uint(tl) << 23) + 0x3F800000u),
            __uint_as_float((__float_as_uint(th) << 23) + 0x3F800000u));
}

}  // namespace qmoe
