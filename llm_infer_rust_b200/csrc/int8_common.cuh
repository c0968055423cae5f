// What the products in 8-bit integers share.
#pragma once
#include <math.h>

#include "common.cuh"

enum : int { INT8_PLAIN = 0, INT8_GLU = 1 };

struct Int8ProductParams {
  const int8_t* q;           // [tokens, k], rows q_pitch bytes apart
  const float* s;            // [tokens]
  const int8_t* w;           // [rows, k], rows w_pitch bytes apart
  const float* c;            // [rows]
  const float* bias;         // [rows] or null
  void* out;                 // [tokens, n]
  int tokens, n, k;          // n: columns of out (INT8_GLU: w has 2 n rows)
  long long q_pitch, w_pitch;
  float limit, alpha;
  int* err;
};

// The device that a call runs on.
struct Int8Device { int index, sms; };

// A kernel's limit of dynamic shared memory is a device's own: set at its first launch on each (beyond 64 devices at every launch).
template <typename Kernel> static int int8_launch_limit(Kernel kernel, int bytes, const Int8Device& device, bool (&set)[64]) {
  const bool kept = device.index >= 0 && device.index < 64;
  if (kept && set[device.index]) return 0;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && kept) set[device.index] = true;
  return static_cast<int>(e);
}

// g / (1 + exp(x)).
// EXACT, for results in float32: good to 8 units of 2^-24 (4.8 at most among 56 million; the fast functions 65), and without a branch: those of
// expf and of a true quotient keep the elements of a row from overlapping (45 tokens at 2 x 12,288 x 4,096 34.2 us so, 23.7 this way and with the fast
// functions; 8,192 at 2 x 2,816 x 1,024 89 us, so 62).
//   exponential   2^p with p = x log2(e) rounded.  What the rounding left, e (by a fused multiply-add, log2(e) in two floats), makes it
//                 2^(p + e) = 2^p (1 + e ln 2) to second order.
//   quotient      times the hardware's reciprocal behind a Newton step.
// Results in bfloat16 take the fast exponential and quotient: 2 + 1.173 |x| units in the last place at an exponent of x, so 2^-18 of the result
// at 16 and 2^-16 at 87, far below their own rounding of 2^-8 (the other way costs them 5 to 10 % where the epilogue bounds: 777 at 2 x 2,816 x
// 1,024 12.4 us, so 13.0).  From an exponent of about 87.3 on, where the factor is below 2e-36, both give 0.
template <bool EXACT> __device__ __forceinline__ float gate_over(float g, float x) {
  if constexpr (EXACT) {
    const float at = fminf(fmaxf(x, -100.0f), 88.5f);  // (beyond: 1 and 0 all the same, and every step stays finite; a NaN comes back with g)
    const float p = __fmul_rn(at, 1.44269502f), e = fmaf(at, 1.92596299e-8f, fmaf(at, 1.44269502f, -p));
    float t, y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(t) : "f"(p));
    const float d = 1.0f + fmaf(t, e * 0.693147181f, t);
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(d));
    return g * fmaf(fmaf(-d, y, 1.0f), y, y);
  } else {
    return __fdividef(g, 1.0f + __expf(x));
  }
}
// What joins gate and up (see glu_product of common.cuh for the forms), each a factor over 1 + exp: tanh(z) = 2 / (1 + exp(-2 z)) - 1.
template <bool EXACT> __device__ __forceinline__ float gate_up(float g, float u, float limit, float alpha) {
#if defined(GLU_CLAMPED_SWISH)
  g = g > limit ? limit : g;                          // (comparisons, not minima: NaN stays)
  u = (u > limit ? limit : u < -limit ? -limit : u) + 1.0f;
  return gate_over<EXACT>(g, -alpha * g) * u;
#elif defined(GLU_GELU_TANH)
  return gate_over<EXACT>(g, -1.5957691216057308f * (g + 0.044715f * g * g * g)) * u;
#else
  return gate_over<EXACT>(g, -g) * u;
#endif
}
