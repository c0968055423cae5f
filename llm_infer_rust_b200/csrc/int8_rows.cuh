// Rows to 8 bits, one scale a row, optionally behind a residual add and an RMS norm.
//
//   a = max_k |x_k|,  s = a / 127,  q_k = rint(x_k * (127 / a))                 (ties to even; float throughout)
//
// With a norm in front, y_k = v_k f g_k with v = x + residual (float, not rounded), f = rsqrt(mean v^2 + eps): the factor f is
// common to the row, so q_k = rint(v_k g_k * (127 / max |v g|)) and s = f max |v g| / 127.  The sum of squares and the
// maximum come out of ONE reduction, and the row is read once.  round(v) is stored as the new residual.
//
// A row of zeros has s = 0 and q = 0.  A row that holds a NaN or an infinity has no 8-bit form: its scale is NaN and its
// q are 0, so everything computed from the row is NaN.  Where 127 / a would overflow (a < 2^-100) row and maximum are
// multiplied by 2^100 first, which is exact.
//
// Bound by the bytes of x (and the residual, twice), by latency where rows are few.  One block a row, the row in registers
// (up to 32 elements a thread) between the reduction and the rounding.
#pragma once
#include "common.cuh"

struct Int8RowsParams {
  const void* x;             // [tokens, k], rows x_pitch elements apart
  const void* residual;      // [tokens, k] or null (in x's type)
  const void* gain;          // [k]: the norm's weight, or null (no norm)
  void* sum_out;             // [tokens, k] or null: round(x + residual)
  int8_t* q;                 // [tokens, k], rows q_pitch bytes apart (a multiple of 16)
  float* s;                  // [tokens]
  int tokens, k;
  long long x_pitch, q_pitch;
  float eps;
  int wide;                  // whether 8 elements of x, residual, gain and sum_out may be moved at once
};

// N = 8 consecutive elements from `p` on (`n` of them exist, the others read as 0).
template <typename T> __device__ __forceinline__ void int8_fetch8(const T* p, int n, bool wide, float (&v)[8]) {
  if (wide && n >= 8) {
    load_floats<T, 8>(p, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? to_f32<T>(p[e]) : 0.0f;
  }
}
template <typename T> __device__ __forceinline__ void int8_store8(T* p, int n, bool wide, const float (&v)[8]) {
  if (wide && n >= 8) {
    __align__(16) T r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = from_f32<T>(v[e]);
#pragma unroll
    for (int e = 0; e < 8; e += 16 / static_cast<int>(sizeof(T)))
      *reinterpret_cast<uint4*>(p + e) = *reinterpret_cast<const uint4*>(r + e);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = from_f32<T>(v[e]);
  }
}

// What a row's maximum (as bits of a float that is not negative) makes of its elements: q = rint(v * pre * inv).
struct Int8Step {
  float pre, inv, scale;
  bool none;
};
__device__ __forceinline__ Int8Step int8_step(uint32_t top_bits, float factor) {
  const float top = __uint_as_float(top_bits);
  Int8Step t;
  t.none = top_bits == 0u || top_bits >= 0x7f800000u;
  t.pre = top < 7.888609052210118e-31f ? 1.2676506002282294e30f : 1.0f;       // 2^-100, 2^100
  t.inv = t.none ? 0.0f : __fdiv_rn(127.0f, top * t.pre);
  t.scale = top_bits >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : __fmul_rn(__fdiv_rn(top, 127.0f), factor);
  return t;
}
// Four elements as four bytes.  Adding 1.5 * 2^23 leaves the nearest whole number (ties to even) in the low bits.
__device__ __forceinline__ uint32_t int8_pack4(const float* v, const Int8Step& t) {
  uint32_t b[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(__fadd_rn(__fmul_rn(v[e] * t.pre, t.inv), 12582912.0f));
  return t.none ? 0u : __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

constexpr int INT8_ROW_CHUNKS = 4;                    // chunks of 8 elements that a thread keeps

template <typename T, typename TG, bool NORM>
__global__ void __launch_bounds__(512) int8_rows_kernel(const Int8RowsParams P) {
  __shared__ float sums[16];
  __shared__ uint32_t tops[16];
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x, threads = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* x = static_cast<const T*>(P.x) + static_cast<size_t>(row) * P.x_pitch;
  const T* residual = NORM && P.residual ? static_cast<const T*>(P.residual) + static_cast<size_t>(row) * P.k : nullptr;
  T* sum_out = NORM && P.sum_out ? static_cast<T*>(P.sum_out) + static_cast<size_t>(row) * P.k : nullptr;
  const TG* gain = static_cast<const TG*>(P.gain);
  const int chunks = (P.k + 7) / 8;
  const bool wide = P.wide != 0, kept = chunks <= INT8_ROW_CHUNKS * threads;

  // v (behind a norm: v * gain) of one chunk; `first`: also the sum's store and the row's sum of squares
  float ss = 0.0f;
  uint32_t top = 0u;
  auto fetch = [&](int c, float (&v)[8], bool first) {
    const int at = c * 8, n = P.k - at;
    int8_fetch8<T>(x + at, n, wide, v);
    if (NORM) {
      if (residual) {
        float r[8];
        int8_fetch8<T>(residual + at, n, wide, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __fadd_rn(v[e], r[e]);
        if (first && sum_out) int8_store8<T>(sum_out + at, n, wide, v);
      }
      float g[8];
      int8_fetch8<TG>(gain + at, n, wide, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (first) ss = fmaf(v[e], v[e], ss);
        v[e] = __fmul_rn(v[e], g[e]);
      }
    }
    if (first) {
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    }
  };
  float v[INT8_ROW_CHUNKS][8];
  if (kept) {
#pragma unroll
    for (int i = 0; i < INT8_ROW_CHUNKS; ++i)
      if (threadIdx.x + i * threads < chunks) fetch(threadIdx.x + i * threads, v[i], true);
  } else {
    for (int c = threadIdx.x; c < chunks; c += threads) fetch(c, v[0], true);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (NORM) ss = warp_sum(ss);
  if (lane == 0) { tops[warp] = top; sums[warp] = ss; }
  __syncthreads();
  top = 0u;
  ss = 0.0f;
  for (int w = 0; w < threads / 32; ++w) {
    top = max(top, tops[w]);
    ss += sums[w];
  }
  const Int8Step step = int8_step(top, NORM ? rsqrtf(ss / static_cast<float>(P.k) + P.eps) : 1.0f);
  if (threadIdx.x == 0) P.s[row] = step.scale;
  int8_t* q = P.q + static_cast<size_t>(row) * P.q_pitch;
  if (kept) {
#pragma unroll
    for (int i = 0; i < INT8_ROW_CHUNKS; ++i)
      if (threadIdx.x + i * threads < chunks)
        *reinterpret_cast<uint2*>(q + (threadIdx.x + i * threads) * 8) = make_uint2(int8_pack4(v[i], step), int8_pack4(v[i] + 4, step));
  } else {
    for (int c = threadIdx.x; c < chunks; c += threads) {
      fetch(c, v[0], false);
      *reinterpret_cast<uint2*>(q + c * 8) = make_uint2(int8_pack4(v[0], step), int8_pack4(v[0] + 4, step));
    }
  }
}

template <typename T>
static int int8_rows_typed(const Int8RowsParams& P, int gain_code, cudaStream_t stream) {
  const int chunks = (P.k + 7) / 8;
  int threads = (chunks + 1) / 2;                       // two chunks a thread: the row's latency, not its issue, is the time
  threads = threads < 32 ? 32 : threads > 512 ? 512 : (threads + 31) / 32 * 32;
  auto kernel = P.gain == nullptr ? int8_rows_kernel<T, float, false>
                : gain_code == B200_F32 ? int8_rows_kernel<T, float, true> : int8_rows_kernel<T, __nv_bfloat16, true>;
  return b200_launch(kernel, dim3(P.tokens), dim3(threads), 0, stream, 0, P);
}
static int int8_rows_launch(const Int8RowsParams& P, int x_code, int gain_code, cudaStream_t stream) {
  if (x_code == B200_F32) return int8_rows_typed<float>(P, gain_code, stream);
  if (x_code == B200_BF16) return int8_rows_typed<__nv_bfloat16>(P, gain_code, stream);
  return B200_BAD_DTYPE;
}
static inline bool int8_aligned(const void* p, long long pitch_bytes) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && pitch_bytes % 16 == 0;
}
