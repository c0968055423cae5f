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

// What joins gate and up (see glu_product of common.cuh for the forms), each a factor over 1 + exp: tanh(z) = 2 / (1 + exp(-2 z)) - 1.
// The fast exponential and quotient are off by a few 2^-22, without the branches of the exact ones, which keep the
// elements of a row from overlapping (a tile of 128 x 128 took 7 us with them, more than its products).
__device__ __forceinline__ float gate_up(float g, float u, float limit, float alpha) {
#if defined(GLU_CLAMPED_SWISH)
  g = g > limit ? limit : g;                          // (comparisons, not minima: NaN stays)
  u = (u > limit ? limit : u < -limit ? -limit : u) + 1.0f;
  return __fdividef(g, 1.0f + __expf(-alpha * g)) * u;
#elif defined(GLU_GELU_TANH)
  return __fdividef(g, 1.0f + __expf(-1.5957691216057308f * (g + 0.044715f * g * g * g))) * u;
#else
  return __fdividef(g, 1.0f + __expf(-g)) * u;
#endif
}
