// Arithmetic that the softmax kernels share (lev_attn_tc.cu, lev_logprobs.cu): two f32 operations per instruction, each
// rounded as on its own, the hardware's power of two and maxima of three.
#pragma once
#include <cuda_runtime.h>

namespace {

typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 two(float lo, float hi) {
    f32x2 v;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ f32x2 twice(float v) { return two(v, v); }
__device__ __forceinline__ void both(f32x2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 fma_2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ f32x2 add_2(f32x2 a, f32x2 b) {
    f32x2 v;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ f32x2 mul_2(f32x2 a, f32x2 b) {
    f32x2 v;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
// 2^x, relative error 2^-22 (the rounding of x comes on top), 0 for -inf
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// 1 / x, relative error 2^-23, 0 for inf
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// a NaN among the three is passed over
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// 2^x for -127 <= x <= 127 on the multiply-add units, for part of the weights where the special function unit (a quarter of their
// rate) bounds a kernel: x = n + f with |f| <= 1/2 by adding and subtracting 1.5 * 2^23, a cubic in f of least maximal relative
// error (Remez's exchange: 7.5e-5, about a sixth of f16's half step), times 2^n from n's bits.  The product is 0 at n = -127, what callers
// clamp lower values to: a weight of 0 is 0, not a least number that bf16 could still represent.  NaN stays NaN.
__device__ __forceinline__ f32x2 exp2_cubic(f32x2 x) {
    const f32x2 r = add_2(x, twice(12582912.f)), f = fma_2(add_2(r, twice(-12582912.f)), twice(-1.f), x);
    f32x2 p = fma_2(f, twice(0.0551716685295105f), twice(0.2426111251115799f));
    p = fma_2(f, p, twice(0.6932609677314758f));
    p = fma_2(f, p, twice(0.9999280571937561f));
    float ra, rb;
    both(r, ra, rb);
    return mul_2(p, two(__uint_as_float(0x3F800000u + (__float_as_uint(ra) << 23)), __uint_as_float(0x3F800000u + (__float_as_uint(rb) << 23))));
}
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if one is NaN
    float y;
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

}  // namespace
