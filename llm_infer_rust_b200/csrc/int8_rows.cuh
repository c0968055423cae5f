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
// Bound by the bytes of x (and the residual, twice), by latency where rows are few.  A block walks over rows; a row lies in
// registers (up to 32 elements a thread) between the reduction and the rounding, the next row's loads are on their way
// meanwhile.  All loads of a row are issued before its first store: a store that might alias would else hold the loads behind it.
#pragma once
#include <string.h>

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

// Eight consecutive elements as they lie in memory.
template <typename T> struct Int8Raw { uint4 v[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ T int8_zero();
template <> __device__ __forceinline__ float int8_zero<float>() { return 0.0f; }
template <> __device__ __forceinline__ __nv_bfloat16 int8_zero<__nv_bfloat16>() { return __float2bfloat16_rn(0.0f); }

// The elements from `p` on, of which `n` exist (the others read as 0).
template <typename T> __device__ __forceinline__ void int8_load8(const T* p, int n, bool wide, Int8Raw<T>& r) {
  if (wide && n >= 8) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < n ? p[i] : int8_zero<T>();
    memcpy(&r, e, sizeof(r));
  }
}
template <typename T> __device__ __forceinline__ void int8_floats(const Int8Raw<T>& r, float (&v)[8]) {
  const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    const uint32_t u[4] = {r.v[sizeof(T) / 2 - 1].x, r.v[sizeof(T) / 2 - 1].y, r.v[sizeof(T) / 2 - 1].z, r.v[sizeof(T) / 2 - 1].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = __uint_as_float(w[i]);
      v[4 + i] = __uint_as_float(u[i]);
    }
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
  if (t.pre == 1.0f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(__fadd_rn(__fmul_rn(v[e], t.inv), 12582912.0f));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(__fadd_rn(__fmul_rn(v[e] * t.pre, t.inv), 12582912.0f));
  }
  return t.none ? 0u : __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

constexpr int INT8_ROW_CHUNKS = 4;                    // chunks of 8 elements that a thread keeps

// The larger of a row's maximum and |v|, NaN if either is.
__device__ __forceinline__ float int8_top(float top, float v) {
  asm("max.NaN.f32 %0, %0, %1;\n" : "+f"(top) : "f"(fabsf(v)));
  return top;
}
// One chunk behind its loads: v = x, or behind a norm (x + residual) * gain, with what it adds to the row's sum of squares and
// maximum; the sum is stored where sum_out is given (`n` of the elements exist).
template <typename T, typename TG, bool NORM>
__device__ __forceinline__ void int8_chunk(const Int8Raw<T>& x, const Int8Raw<T>& r, const Int8Raw<TG>& gain, bool add, T* sum_out, int n,
                                           bool wide, float (&v)[8], float& ss, float& top) {
  int8_floats<T>(x, v);
  if (NORM) {
    float f[8];
    if (add) {
      int8_floats<T>(r, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __fadd_rn(v[e], f[e]);
      if (sum_out) int8_store8<T>(sum_out, n, wide, v);
    }
    int8_floats<TG>(gain, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ss = fmaf(v[e], v[e], ss);
      v[e] = __fmul_rn(v[e], f[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) top = int8_top(top, v[e]);
}

// The block's sums of squares and maximum (`turn`: which half of the scratch is free).
// Returns the maximum's bits: as integers floats that are not negative compare as they do, and NaN is above infinity.
template <bool NORM> __device__ __forceinline__ uint32_t int8_meet(float& ss, float top, float (*sums)[32], uint32_t (*tops)[32], int turn) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  if (NORM) ss = warp_sum(ss);
  if (lane == 0) { tops[turn][warp] = bits; sums[turn][warp] = ss; }
  __syncthreads();
  if (NORM) {
    ss = 0.0f;
    for (int w = 0; w < warps; ++w) ss += sums[turn][w];
  }
  return __reduce_max_sync(0xffffffffu, lane < warps ? tops[turn][lane] : 0u);
}

// Rows whose chunks fit the block's registers, CH a thread.
template <typename T, typename TG, bool NORM, int CH, int MOST = 512>
__global__ void __launch_bounds__(MOST) int8_rows_kernel(const Int8RowsParams P) {
  __shared__ float sums[2][32];
  __shared__ uint32_t tops[2][32];
  pdl_launch_dependents();
  pdl_wait();
  const int threads = blockDim.x, chunks = (P.k + 7) / 8;
  const bool wide = P.wide != 0, add = NORM && P.residual != nullptr;
  const TG* gain = static_cast<const TG*>(P.gain);
  constexpr int AHEAD = 1;
  Int8Raw<T> x[AHEAD][CH], r[AHEAD][CH];
  auto load = [&](int row, Int8Raw<T> (&x)[CH], Int8Raw<T> (&r)[CH]) {
    if (row >= P.tokens) return;
    const T* xs = static_cast<const T*>(P.x) + static_cast<size_t>(row) * P.x_pitch;
    const T* rs = static_cast<const T*>(P.residual) + static_cast<size_t>(row) * P.k;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int at = (threadIdx.x + i * threads) * 8;
      if (at >= P.k) continue;
      int8_load8<T>(xs + at, P.k - at, wide, x[i]);
      if (add) int8_load8<T>(rs + at, P.k - at, wide, r[i]);
    }
  };
  int turn = 0;
  auto take = [&](int row, Int8Raw<T> (&x)[CH], Int8Raw<T> (&r)[CH]) {
    Int8Raw<TG> g[CH];
    if (NORM)
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int at = (threadIdx.x + i * threads) * 8;
        if (at < P.k) int8_load8<TG>(gain + at, P.k - at, wide, g[i]);
      }
    T* sum_out = add && P.sum_out ? static_cast<T*>(P.sum_out) + static_cast<size_t>(row) * P.k : nullptr;
    float v[CH][8], ss = 0.0f;
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int at = (threadIdx.x + i * threads) * 8;
      if (at < P.k) int8_chunk<T, TG, NORM>(x[i], r[i], g[i], add, sum_out ? sum_out + at : nullptr, P.k - at, wide, v[i], ss, top);
    }
    load(row + AHEAD * gridDim.x, x, r);
    const uint32_t bits = int8_meet<NORM>(ss, top, sums, tops, turn);
    turn ^= 1;
    const Int8Step step = int8_step(bits, NORM ? rsqrtf(ss / static_cast<float>(P.k) + P.eps) : 1.0f);
    if (threadIdx.x == 0) P.s[row] = step.scale;
    int8_t* q = P.q + static_cast<size_t>(row) * P.q_pitch;
#pragma unroll
    for (int i = 0; i < CH; ++i)
      if (threadIdx.x + i * threads < chunks)
        *reinterpret_cast<uint2*>(q + (threadIdx.x + i * threads) * 8) = make_uint2(int8_pack4(v[i], step), int8_pack4(v[i] + 4, step));
  };
#pragma unroll
  for (int a = 0; a < AHEAD; ++a) load(blockIdx.x + a * gridDim.x, x[a], r[a]);
  for (int row = blockIdx.x; row < P.tokens; row += AHEAD * gridDim.x)
#pragma unroll
    for (int a = 0; a < AHEAD; ++a)
      if (row + a * static_cast<int>(gridDim.x) < P.tokens) take(row + a * gridDim.x, x[a], r[a]);
}

// Many long bfloat16 rows without a norm: eight chunks a thread, kept AS THEY LIE IN MEMORY and taken apart once for the maximum and
// once for the rounding.  With two chunks a thread, what every thread does once a row (the reduction, the division, addresses) was
// two thirds of 15 instructions an element and bound the kernel: 8,192 x 4,096 20.4 -> 17.1 us (5.9 TB/s), 8,192 x 12,288 64 -> 47 us
// (6.4 TB/s).  Short rows and few rows lose by it (8,192 x 1,024 6.7 -> 9.0 us, 300 x 4,096 2.5 -> 2.8), rows behind a norm too, whose
// two inputs leave room for few threads (8,192 x 4,096 45 -> 47 us).
template <typename T>
__global__ void __launch_bounds__(256) int8_many_rows_kernel(const Int8RowsParams P) {
  constexpr int CH = 8;
  __shared__ float sums[1][32];
  __shared__ uint32_t tops[1][32];
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x, threads = blockDim.x;
  const T* xs = static_cast<const T*>(P.x) + static_cast<size_t>(row) * P.x_pitch;
  Int8Raw<T> x[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int at = (threadIdx.x + i * threads) * 8;
    if (at < P.k) int8_load8<T>(xs + at, 8, true, x[i]);        // (whole chunks: the launch sees to it)
  }
  float v[8], ss = 0.0f, top = 0.0f;
#pragma unroll
  for (int i = 0; i < CH; ++i)
    if ((threadIdx.x + i * threads) * 8 < P.k) {
      int8_floats<T>(x[i], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = int8_top(top, v[e]);
    }
  const Int8Step step = int8_step(int8_meet<false>(ss, top, sums, tops, 0), 1.0f);
  if (threadIdx.x == 0) P.s[row] = step.scale;
  int8_t* q = P.q + static_cast<size_t>(row) * P.q_pitch;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int at = (threadIdx.x + i * threads) * 8;
    if (at < P.k) {
      int8_floats<T>(x[i], v);
      *reinterpret_cast<uint2*>(q + at) = make_uint2(int8_pack4(v, step), int8_pack4(v + 4, step));
    }
  }
}

// Longer rows are read twice.
template <typename T, typename TG, bool NORM>
__global__ void __launch_bounds__(512) int8_long_rows_kernel(const Int8RowsParams P) {
  __shared__ float sums[1][32];
  __shared__ uint32_t tops[1][32];
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x, chunks = (P.k + 7) / 8;
  const bool wide = P.wide != 0, add = NORM && P.residual != nullptr;
  const T* xs = static_cast<const T*>(P.x) + static_cast<size_t>(row) * P.x_pitch;
  const T* rs = static_cast<const T*>(P.residual) + static_cast<size_t>(row) * P.k;
  const TG* gain = static_cast<const TG*>(P.gain);
  T* sum_out = add && P.sum_out ? static_cast<T*>(P.sum_out) + static_cast<size_t>(row) * P.k : nullptr;
  float ss = 0.0f;
  float top = 0.0f;
  auto fetch = [&](int c, float (&v)[8], T* store) {
    const int at = c * 8;
    Int8Raw<T> x, r;
    Int8Raw<TG> g;
    int8_load8<T>(xs + at, P.k - at, wide, x);
    if (add) int8_load8<T>(rs + at, P.k - at, wide, r);
    if (NORM) int8_load8<TG>(gain + at, P.k - at, wide, g);
    int8_chunk<T, TG, NORM>(x, r, g, add, store ? store + at : nullptr, P.k - at, wide, v, ss, top);
  };
  for (int c = threadIdx.x; c < chunks; c += blockDim.x) {
    float v[8];
    fetch(c, v, sum_out);
  }
  const uint32_t bits = int8_meet<NORM>(ss, top, sums, tops, 0);
  const Int8Step step = int8_step(bits, NORM ? rsqrtf(ss / static_cast<float>(P.k) + P.eps) : 1.0f);
  if (threadIdx.x == 0) P.s[row] = step.scale;
  int8_t* q = P.q + static_cast<size_t>(row) * P.q_pitch;
  for (int c = threadIdx.x; c < chunks; c += blockDim.x) {
    float v[8];
    fetch(c, v, nullptr);
    *reinterpret_cast<uint2*>(q + c * 8) = make_uint2(int8_pack4(v, step), int8_pack4(v + 4, step));
  }
}

template <typename T, typename TG, bool NORM, int CH, int MOST = 512>
static int int8_rows_kept(const Int8RowsParams& P, int threads, int sms, cudaStream_t stream) {
  // Persistent: as many blocks as fit at once (threads, registers: found once for each size of block).
  static int fits[33];
  int& blocks = fits[threads / 32];
  if (blocks == 0) {
    int n = 0;
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, int8_rows_kernel<T, TG, NORM, CH, MOST>, threads, 0);
    if (e != cudaSuccess) return static_cast<int>(e);
    blocks = n < 1 ? 1 : n;
  }
  const int most = sms * blocks;
  return b200_launch(int8_rows_kernel<T, TG, NORM, CH, MOST>, dim3(P.tokens < most ? P.tokens : most), dim3(threads), 0, stream, 0, P);
}
template <typename T, typename TG, bool NORM>
static int int8_rows_normed(const Int8RowsParams& P, int sms, cudaStream_t stream) {
  const int chunks = (P.k + 7) / 8;
  auto threads = [&](int ch) { return ((chunks + ch - 1) / ch + 31) / 32 * 32; };
  if constexpr (sizeof(T) == 2 && !NORM)
    if (P.tokens > 8 * sms && P.wide && P.k % 8 == 0 && chunks >= 512 && chunks <= 2048)
      return b200_launch(int8_many_rows_kernel<T>, dim3(P.tokens), dim3(threads(8)), 0, stream, 0, P);
  // Few rows: the row's latency is the time, so a thread takes as little as 512 of them allow.  Many: what counts are the bytes on
  // their way; two chunks a thread keep them (8,192 x 4,096 behind a norm 45 us; four chunks, half the threads: 61), and rows longer
  // than that are faster read twice, the second time out of the caches (8,192 x 12,288 behind a norm 130 us, 5.4 TB/s), but for float32
  // without a norm, where 1,024 threads still keep theirs (2,048 x 12,288: 20 us, read twice 25).
  if (P.tokens <= sms) {
    if (chunks <= 512) return int8_rows_kept<T, TG, NORM, 1>(P, threads(1), sms, stream);
    if (chunks <= 1024) return int8_rows_kept<T, TG, NORM, 2>(P, threads(2), sms, stream);
    if (chunks <= 512 * INT8_ROW_CHUNKS) return int8_rows_kept<T, TG, NORM, INT8_ROW_CHUNKS>(P, threads(INT8_ROW_CHUNKS), sms, stream);
  } else if (chunks <= 1024) {
    return int8_rows_kept<T, TG, NORM, 2>(P, threads(2), sms, stream);
  } else if (!NORM && sizeof(T) == 4 && chunks <= 2048) {
    return int8_rows_kept<T, TG, false, 2, 1024>(P, threads(2), sms, stream);
  }
  return b200_launch(int8_long_rows_kernel<T, TG, NORM>, dim3(P.tokens), dim3(512), 0, stream, 0, P);
}
template <typename T>
static int int8_rows_typed(const Int8RowsParams& P, int gain_code, int sms, cudaStream_t stream) {
  if (P.gain == nullptr) return int8_rows_normed<T, float, false>(P, sms, stream);
  return gain_code == B200_F32 ? int8_rows_normed<T, float, true>(P, sms, stream) : int8_rows_normed<T, __nv_bfloat16, true>(P, sms, stream);
}
static int int8_rows_launch(const Int8RowsParams& P, int x_code, int gain_code, int sms, cudaStream_t stream) {
  if (x_code == B200_F32) return int8_rows_typed<float>(P, gain_code, sms, stream);
  if (x_code == B200_BF16) return int8_rows_typed<__nv_bfloat16>(P, gain_code, sms, stream);
  return B200_BAD_DTYPE;
}
static inline bool int8_aligned(const void* p, long long pitch_bytes) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && pitch_bytes % 16 == 0;
}
