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
// Bound by the bytes of x (and the residual, twice), by latency where rows are few.  A block (short rows: a warp) walks over rows; a
// row lies in registers (up to 32 elements a thread) between the reduction and the rounding, the next row's loads are on their way
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
  int whole;                 // whether every row of x, residual, gain and sum_out is whole eights of elements at multiples of 16 bytes
};

// Eight consecutive elements as they lie in memory.
template <typename T> struct Int8Raw { uint4 v[sizeof(T) / 2]; };

// The words w[0 .. N) of what begins `bytes` (an even number below 20) behind w's start.  (Branches on a number that all threads
// share: word by word selections cost three times the instructions.)
template <int BY, int N, int M> __device__ __forceinline__ void int8_shift_by(uint32_t (&w)[M], uint32_t bits) {
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = i + BY + 1 < M ? __funnelshift_r(w[i + BY], w[i + BY + 1], bits) : w[i + BY] >> bits;
}
template <int N, int M> __device__ __forceinline__ void int8_shift(uint32_t (&w)[M], int bytes) {
  const uint32_t bits = (bytes & 2) * 8;
  switch (bytes >> 2) {
    case 0: int8_shift_by<0, N>(w, bits); break;
    case 1: int8_shift_by<1, N>(w, bits); break;
    case 2: int8_shift_by<2, N>(w, bits); break;
    case 3: int8_shift_by<3, N>(w, bits); break;
    default: int8_shift_by<4, N>(w, bits); break;
  }
}

// Eight elements in a row from `p` on, of which `n` exist (the others read as 0).  WHOLE: all of them do, at a multiple of 16 bytes.
// Else the aligned 16-byte pieces that hold them are fetched and shifted into place: rows whose length is no multiple of eight begin
// anywhere, and element by element they took three times as long.  (No piece without an element of the row is touched: of the eight
// the first `lead` do not exist either; what they read as is the caller's affair.)
template <typename T, bool WHOLE> __device__ __forceinline__ void int8_load8(const T* p, int n, Int8Raw<T>& r, int lead = 0) {
  constexpr int PIECES = sizeof(T) / 2;
  if constexpr (WHOLE) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15u), bytes = off + min(n, 8) * static_cast<int>(sizeof(T));
    const uint4* from = reinterpret_cast<const uint4*>(p - off / static_cast<int>(sizeof(T)));
    if (off == 0 && n >= 8 && lead == 0) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) r.v[i] = from[i];
      return;
    }
    uint32_t w[PIECES * 4 + 5];
#pragma unroll
    for (int i = 0; i <= PIECES; ++i) {
      const bool any = i * 16 < bytes && i * 16 + 16 > off + lead * static_cast<int>(sizeof(T));
      const uint4 v = any ? from[i] : make_uint4(0u, 0u, 0u, 0u);
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
    w[PIECES * 4 + 4] = 0u;
    int8_shift<PIECES * 4, PIECES * 4 + 5>(w, off);
    if (n < 8) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (sizeof(T) == 2) {
          if (e >= n) w[e / 2] &= e % 2 ? 0x0000ffffu : 0u;
        } else {
          if (e >= n) w[e] = 0u;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) r.v[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
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
// Eight floats as T, in words.
template <typename T> __device__ __forceinline__ void int8_words(const float (&v)[8], uint32_t (&w)[sizeof(T) * 2]) {
#pragma unroll
  for (int e = 0; e < static_cast<int>(sizeof(T)) * 2; ++e) {
    if constexpr (sizeof(T) == 2) {
      const __nv_bfloat162 pair = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
      memcpy(&w[e], &pair, 4);
    } else {
      w[e] = __float_as_uint(v[e]);
    }
  }
}
// The chunk at column `at` of a row of k elements.  WHOLE: as in int8_load8.  Else every lane of the warp calls (those beyond the row
// store nothing): where the row begins off a multiple of 16 bytes, a lane stores the aligned pieces that begin in the chunk before,
// with that lane's last bytes in front; the pieces at the ends of the warp's stretch are stored element by element.
template <typename T, bool WHOLE> __device__ __forceinline__ void int8_store8(T* row, int at, int k, const float (&v)[8]) {
  constexpr int N = sizeof(T) * 2, SIZE = sizeof(T);
  uint32_t w[N];
  int8_words<T>(v, w);
  if constexpr (WHOLE) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<uint4*>(row + at + i * 4 / SIZE) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  } else {
    const int lane = threadIdx.x & 31, off = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15u), n = k - at;
    if (off == 0) {                                             // (all lanes' rows are this one)
      if (n >= 8) return int8_store8<T, true>(row, at, k, v);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) row[at + e] = from_f32<T>(v[e]);
      return;
    }
    uint32_t c[N + 5];                                          // the chunk before this one's last 16 bytes, then this one
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = __shfl_up_sync(0xffffffffu, w[N - 4 + i], 1);
#pragma unroll
    for (int i = 0; i < N; ++i) c[4 + i] = w[i];
    c[N + 4] = 0u;
    int8_shift<N, N + 5>(c, 16 - off);                          // to the first aligned piece
    T* aligned = row + at - off / SIZE;
    const bool full = n >= 8, joins = full && lane > 0;               // its first piece lies in two chunks' elements
    const bool joined = lane < 31 && n >= 16;                                       // ... and so does what is behind its last
    if (joins) *reinterpret_cast<uint4*>(aligned) = make_uint4(c[0], c[1], c[2], c[3]);
    if (full && N == 8) *reinterpret_cast<uint4*>(aligned + 16 / SIZE) = make_uint4(c[N - 4], c[N - 3], c[N - 2], c[N - 1]);
    const int head = (16 - off) / SIZE, tail = 8 - off / SIZE;
    if (!joins || !joined) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n && ((!joins && (!full || e < head)) || (full && !joined && e >= tail))) row[at + e] = from_f32<T>(v[e]);
    }
  }
}

// Rows that are not whole, AS THEY LIE: a thread's eight elements begin at a multiple of 16 bytes, so at columns c, c + 8, ... with
// -16 bytes < c <= 0, and nothing is shifted on its way in or out but the gain (which lies otherwise to every row) and the 8-bit
// results, that begin at a multiple of 16 bytes in every row.  With x, the residual and the sum shifted to columns 0, 8, ... the
// instructions bound the kernel: 8,192 x 1,999 bfloat16 behind a norm 46.5 -> 28.0 us (3.8 TB/s; whole rows of 2,000 20), float32
// 69 -> 44, 4,042 x 4,407 55 -> 35, without a norm 17.5 -> 15.5.

// How many elements lie between the multiple of 16 bytes at or before p and p.
template <typename T, bool WHOLE> __device__ __forceinline__ int int8_lead(const T* p) {
  return WHOLE ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15u) / static_cast<int>(sizeof(T));
}
// Columns c .. c + 8 of a row of k elements (those that are none are read as anything; int8_trim).  LIES: row + c is a multiple of 16
// bytes.
template <typename T, bool WHOLE, bool LIES = true> __device__ __forceinline__ void int8_fetch(const T* row, int c, int k, Int8Raw<T>& r) {
  constexpr int PIECES = sizeof(T) / 2, PER = 16 / sizeof(T);
  if constexpr (WHOLE) {
    int8_load8<T, true>(row + c, 8, r);
  } else {
    if (LIES || c >= k) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) r.v[i] = c + i * PER < k ? reinterpret_cast<const uint4*>(row + c)[i] : make_uint4(0u, 0u, 0u, 0u);
    } else {
      int8_load8<T, false>(row + c, k - c, r, max(-c, 0));
    }
  }
}
// What lies beside the row becomes 0.
template <bool WHOLE> __device__ __forceinline__ void int8_trim(float (&v)[8], int c, int k) {
  if (!WHOLE && (c < 0 || c + 8 > k)) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (static_cast<unsigned>(c + e) >= static_cast<unsigned>(k)) v[e] = 0.0f;
  }
}
// Columns c .. c + 8 as they go out, rounded to T.
template <typename T, bool WHOLE> __device__ __forceinline__ void int8_put_sum(T* row, int c, int k, const float (&v)[8]) {
  constexpr int PIECES = sizeof(T) / 2, PER = 16 / sizeof(T);
  if constexpr (WHOLE) {
    int8_store8<T, true>(row, c, k, v);
  } else {
    const bool lies = (reinterpret_cast<uintptr_t>(row + c) & 15u) == 0;
    uint32_t w[sizeof(T) * 2];
    int8_words<T>(v, w);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = c + i * PER;
      if (lies && at >= 0 && at + PER <= k) {
        reinterpret_cast<uint4*>(row + c)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      } else {
#pragma unroll
        for (int e = 0; e < PER; ++e)
          if (at + e >= 0 && at + e < k) row[at + e] = from_f32<T>(v[i * PER + e]);
      }
    }
  }
}
// A thread's column in its i-th chunk of CH: not WHOLE, a warp's chunks follow one another.
template <bool WHOLE, int CH> __device__ __forceinline__ int int8_column(int i, int lead) {
  return WHOLE ? static_cast<int>(threadIdx.x + i * blockDim.x) * 8
               : static_cast<int>((threadIdx.x & ~31u) * CH + i * 32 + (threadIdx.x & 31)) * 8 - lead;
}
// Whether a thread (not WHOLE: the whole warp) has nothing at its column c.
template <bool WHOLE> __device__ __forceinline__ bool int8_beyond(int c, int k) {
  return WHOLE ? c >= k : c - static_cast<int>(threadIdx.x & 31) * 8 >= k;
}
// The 8-bit results of a warp's chunks, the first at column c.  Not WHOLE: every lane calls; c + lead is a multiple of eight, a lane
// stores eight results from there on, the last of them the next lane's first, and where two warps meet they go byte by byte.  ALONE:
// the warp has the whole row.
template <int CH, bool ALONE>
__device__ __forceinline__ void int8_put(int8_t* row, int c, int lead, int k, const uint32_t (&low)[CH], const uint32_t (&high)[CH]) {
  const int lane = threadIdx.x & 31;
  const uint32_t bits = (lead & 3) * 8;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int at = c + lead + i * 256;
    const uint32_t low2 = __shfl_sync(0xffffffffu, i + 1 < CH && lane == 0 ? low[i + 1 < CH ? i + 1 : i] : low[i], lane + 1);
    const uint32_t high2 = __shfl_sync(0xffffffffu, i + 1 < CH && lane == 0 ? high[i + 1 < CH ? i + 1 : i] : high[i], lane + 1);
    const uint32_t w0 = lead < 4 ? low[i] : high[i], w1 = lead < 4 ? high[i] : low2, w2 = lead < 4 ? low2 : high2;
    if (at < k && (ALONE || i + 1 < CH || lane < 31 || lead == 0))
      *reinterpret_cast<uint2*>(row + at) = make_uint2(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits));
  }
  if (!ALONE && lead > 0) {
    const bool head = lane < lead;
    const uint32_t l0 = __shfl_sync(0xffffffffu, low[0], 0), h0 = __shfl_sync(0xffffffffu, high[0], 0);
    const uint32_t l1 = __shfl_sync(0xffffffffu, low[CH - 1], 31), h1 = __shfl_sync(0xffffffffu, high[CH - 1], 31);
    const int at = c - lane * 8 + (head ? 0 : CH * 256 - 8) + lane;
    const uint32_t word = lane < 4 ? (head ? l0 : l1) : (head ? h0 : h1);
    if (lane < 8 && at >= 0 && at < k) row[at] = static_cast<int8_t>(word >> (lane & 3) * 8);
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
// One chunk behind its loads: v = x, or behind a residual add x + residual ...
template <typename T> __device__ __forceinline__ void int8_sum(const Int8Raw<T>& x, const Int8Raw<T>& r, bool add, float (&v)[8]) {
  int8_floats<T>(x, v);
  if (add) {
    float f[8];
    int8_floats<T>(r, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __fadd_rn(v[e], f[e]);
  }
}
// ... and what it adds to the row's sum of squares and maximum; behind a norm v becomes v * gain.
template <typename TG, bool NORM, bool WHOLE>
__device__ __forceinline__ void int8_gain(const Int8Raw<TG>& gain, float (&v)[8], int c, int k, float& ss, float& top) {
  if (NORM) {
    float f[8];
    int8_floats<TG>(gain, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ss = fmaf(v[e], v[e], ss);
      v[e] = __fmul_rn(v[e], f[e]);
    }
    int8_trim<WHOLE>(v, c, k);                                  // (what is read beside the gain may be no number)
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) top = int8_top(top, v[e]);
}

// The block's sums of squares and maximum (`turn`: which half of the scratch is free).
// Returns the maximum's bits: as integers floats that are not negative compare as they do, and NaN is above infinity.
template <bool NORM, bool ALONE = false>
__device__ __forceinline__ uint32_t int8_meet(float& ss, float top, float (*sums)[32], uint32_t (*tops)[32], int turn) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  if (NORM) ss = warp_sum(ss);
  if constexpr (ALONE) return bits;
  if (lane == 0) { tops[turn][warp] = bits; sums[turn][warp] = ss; }
  __syncthreads();
  if (NORM) {
    ss = 0.0f;
    for (int w = 0; w < warps; ++w) ss += sums[turn][w];
  }
  return __reduce_max_sync(0xffffffffu, lane < warps ? tops[turn][lane] : 0u);
}

// Rows whose chunks fit the block's registers, CH a thread (ALONE: a warp's, of which a block has blockDim.y).  WHOLE: there are whole
// chunks alone, all at multiples of 16 bytes.
// (8,192 x 4,096 behind a norm with that question asked chunk by chunk 45 us, so 38: 6.2 TB/s, 95 % of the copy rate.)
template <typename T, typename TG, bool NORM, int CH, bool WHOLE, int MOST = 512, bool ALONE = false>
__global__ void __launch_bounds__(MOST) int8_rows_kernel(const Int8RowsParams P) {
  __shared__ float sums[2][32];
  __shared__ uint32_t tops[2][32];
  pdl_launch_dependents();
  pdl_wait();
  const int first = ALONE ? blockIdx.x * blockDim.y + threadIdx.y : blockIdx.x;
  const int step_rows = ALONE ? gridDim.x * blockDim.y : gridDim.x;
  const bool add = NORM && P.residual != nullptr;
  const TG* gain = static_cast<const TG*>(P.gain);
  Int8Raw<T> x[CH], r[CH];
  auto load = [&](int row) {
    if (row >= P.tokens) return;
    const T* xs = static_cast<const T*>(P.x) + static_cast<size_t>(row) * P.x_pitch;
    const T* rs = static_cast<const T*>(P.residual) + static_cast<size_t>(row) * P.k;
    const int lead = int8_lead<T, WHOLE>(xs);
    const bool alike = lead == int8_lead<T, WHOLE>(rs);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = int8_column<WHOLE, CH>(i, lead);
      if (int8_beyond<WHOLE>(c, P.k)) continue;
      int8_fetch<T, WHOLE>(xs, c, P.k, x[i]);
      if (add && alike) int8_fetch<T, WHOLE>(rs, c, P.k, r[i]);
      else if (add) int8_fetch<T, WHOLE, false>(rs, c, P.k, r[i]);
    }
  };
  Int8Raw<TG> g[CH];
  int turn = 0, held = -1;                    // (rows that lie alike need the gain once: the launch sees to it that a block's rows do)
  load(first);
  for (int row = first; row < P.tokens; row += step_rows, turn ^= 1) {
    const int lead = int8_lead<T, WHOLE>(static_cast<const T*>(P.x) + static_cast<size_t>(row) * P.x_pitch);
    if (NORM && (WHOLE || lead != held)) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = int8_column<WHOLE, CH>(i, lead);
        if (!int8_beyond<WHOLE>(c, P.k)) int8_fetch<TG, WHOLE, false>(gain, c, P.k, g[i]);
      }
      held = lead;
    }
    T* sum_out = add && P.sum_out ? static_cast<T*>(P.sum_out) + static_cast<size_t>(row) * P.k : nullptr;
    float v[CH][8], ss = 0.0f, top = 0.0f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = int8_column<WHOLE, CH>(i, lead);
      if (int8_beyond<WHOLE>(c, P.k)) continue;
      int8_sum<T>(x[i], r[i], add, v[i]);
      int8_trim<WHOLE>(v[i], c, P.k);
      if (NORM && sum_out) int8_put_sum<T, WHOLE>(sum_out, c, P.k, v[i]);
      int8_gain<TG, NORM, WHOLE>(g[i], v[i], c, P.k, ss, top);
    }
    load(row + step_rows);
    const uint32_t bits = int8_meet<NORM, ALONE>(ss, top, sums, tops, turn);
    const Int8Step step = int8_step(bits, NORM ? rsqrtf(ss / static_cast<float>(P.k) + P.eps) : 1.0f);
    if (threadIdx.x == 0) P.s[row] = step.scale;
    int8_t* q = P.q + static_cast<size_t>(row) * P.q_pitch;
    uint32_t low[CH], high[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = int8_column<WHOLE, CH>(i, lead);
      low[i] = high[i] = 0u;
      if (int8_beyond<WHOLE>(c, P.k)) continue;
      low[i] = int8_pack4(v[i], step);
      high[i] = int8_pack4(v[i] + 4, step);
      if (WHOLE) *reinterpret_cast<uint2*>(q + c) = make_uint2(low[i], high[i]);
    }
    if (!WHOLE) int8_put<CH, ALONE>(q, int8_column<WHOLE, CH>(0, lead), lead, P.k, low, high);
  }
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
  const int row = blockIdx.x;
  const T* xs = static_cast<const T*>(P.x) + static_cast<size_t>(row) * P.x_pitch;
  Int8Raw<T> x[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = int8_column<true, CH>(i, 0);
    if (!int8_beyond<true>(c, P.k)) int8_fetch<T, true>(xs, c, P.k, x[i]);
  }
  float v[8], ss = 0.0f, top = 0.0f;
#pragma unroll
  for (int i = 0; i < CH; ++i)
    if (!int8_beyond<true>(int8_column<true, CH>(i, 0), P.k)) {
      int8_floats<T>(x[i], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = int8_top(top, v[e]);
    }
  const Int8Step step = int8_step(int8_meet<false>(ss, top, sums, tops, 0), 1.0f);
  if (threadIdx.x == 0) P.s[row] = step.scale;
  int8_t* q = P.q + static_cast<size_t>(row) * P.q_pitch;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = int8_column<true, CH>(i, 0);
    if (int8_beyond<true>(c, P.k)) continue;
    int8_floats<T>(x[i], v);
    *reinterpret_cast<uint2*>(q + c) = make_uint2(int8_pack4(v, step), int8_pack4(v + 4, step));
  }
}

// Longer rows are read twice.
template <typename T, typename TG, bool NORM, bool WHOLE>
__global__ void __launch_bounds__(512) int8_long_rows_kernel(const Int8RowsParams P) {
  __shared__ float sums[1][32];
  __shared__ uint32_t tops[1][32];
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x;
  const bool add = NORM && P.residual != nullptr;
  const T* xs = static_cast<const T*>(P.x) + static_cast<size_t>(row) * P.x_pitch;
  const T* rs = static_cast<const T*>(P.residual) + static_cast<size_t>(row) * P.k;
  const TG* gain = static_cast<const TG*>(P.gain);
  T* sum_out = add && P.sum_out ? static_cast<T*>(P.sum_out) + static_cast<size_t>(row) * P.k : nullptr;
  float ss = 0.0f, top = 0.0f;
  const int lead = int8_lead<T, WHOLE>(xs);
  const bool alike = lead == int8_lead<T, WHOLE>(rs);
  auto fetch = [&](int c, float (&v)[8], bool store) {
    Int8Raw<T> x, r;
    Int8Raw<TG> g;
    int8_fetch<T, WHOLE>(xs, c, P.k, x);
    if (add && alike) int8_fetch<T, WHOLE>(rs, c, P.k, r);
    else if (add) int8_fetch<T, WHOLE, false>(rs, c, P.k, r);
    if (NORM) int8_fetch<TG, WHOLE, false>(gain, c, P.k, g);
    int8_sum<T>(x, r, add, v);
    int8_trim<WHOLE>(v, c, P.k);
    if (NORM && store) int8_put_sum<T, WHOLE>(sum_out, c, P.k, v);
    int8_gain<TG, NORM, WHOLE>(g, v, c, P.k, ss, top);
  };
  for (int c = threadIdx.x * 8 - lead; !int8_beyond<WHOLE>(c, P.k); c += blockDim.x * 8) {
    float v[8];
    fetch(c, v, sum_out != nullptr);
  }
  const uint32_t bits = int8_meet<NORM>(ss, top, sums, tops, 0);
  const Int8Step step = int8_step(bits, NORM ? rsqrtf(ss / static_cast<float>(P.k) + P.eps) : 1.0f);
  if (threadIdx.x == 0) P.s[row] = step.scale;
  int8_t* q = P.q + static_cast<size_t>(row) * P.q_pitch;
  for (int c = threadIdx.x * 8 - lead; !int8_beyond<WHOLE>(c, P.k); c += blockDim.x * 8) {
    float v[8];
    fetch(c, v, false);
    const uint32_t low[1] = {int8_pack4(v, step)}, high[1] = {int8_pack4(v + 4, step)};
    if (WHOLE) *reinterpret_cast<uint2*>(q + c) = make_uint2(low[0], high[0]);
    else int8_put<1, false>(q, c, lead, P.k, low, high);
  }
}

template <typename T, typename TG, bool NORM, int CH, bool WHOLE>
static int int8_rows_warps(const Int8RowsParams& P, int sms, cudaStream_t stream) {
  static int blocks;
  const auto kernel = int8_rows_kernel<T, TG, NORM, CH, WHOLE, 256, true>;
  if (blocks == 0) {
    int n = 0;
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, 256, 0);
    if (e != cudaSuccess) return static_cast<int>(e);
    blocks = n < 1 ? 1 : n;
  }
  const int want = (P.tokens + 7) / 8, most = sms * blocks;
  return b200_launch(kernel, dim3(want < most ? want : most), dim3(32, 8), 0, stream, 0, P);
}
template <typename T, typename TG, bool NORM, int CH, bool WHOLE, int MOST = 512>
static int int8_rows_blocks(const Int8RowsParams& P, int threads, int sms, cudaStream_t stream) {
  // Persistent: as many blocks as fit at once (threads, registers: found once for each size of block).
  static int fits[33];
  int& blocks = fits[threads / 32];
  if (blocks == 0) {
    int n = 0;
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, int8_rows_kernel<T, TG, NORM, CH, WHOLE, MOST>, threads, 0);
    if (e != cudaSuccess) return static_cast<int>(e);
    blocks = n < 1 ? 1 : n;
  }
  const int most = WHOLE ? sms * blocks : sms * blocks & ~7;                    // (rows eight apart lie alike)
  return b200_launch(int8_rows_kernel<T, TG, NORM, CH, WHOLE, MOST>, dim3(P.tokens < most ? P.tokens : most), dim3(threads), 0, stream, 0, P);
}
template <typename T, typename TG, bool NORM, int CH, int MOST = 512>
static int int8_rows_kept(const Int8RowsParams& P, int threads, int sms, cudaStream_t stream) {
  return P.whole ? int8_rows_blocks<T, TG, NORM, CH, true, MOST>(P, threads, sms, stream)
                                : int8_rows_blocks<T, TG, NORM, CH, false, MOST>(P, threads, sms, stream);
}
template <typename T, typename TG, bool NORM>
static int int8_rows_normed(const Int8RowsParams& P, int sms, cudaStream_t stream) {
  const int chunks = (P.k + (P.whole ? 0 : 16 / static_cast<int>(sizeof(T)) - 1) + 7) / 8;
  auto threads = [&](int ch) { return ((chunks + ch - 1) / ch + 31) / 32 * 32; };
  if constexpr (sizeof(T) == 2 && !NORM)
    if (P.tokens > 8 * sms && P.whole && chunks >= 512 && chunks <= 2048)
      return b200_launch(int8_many_rows_kernel<T>, dim3(P.tokens), dim3(threads(8)), 0, stream, 0, P);
  // Few rows: the row's latency is the time, so a thread takes as little as 512 of them allow.  Many: what counts are the bytes on
  // their way; two chunks a thread keep them (behind a norm 8,192 x 4,096 38 us; four chunks, half the threads: a third slower), in up
  // to 1,024 threads (8,192 x 12,288 bfloat16 behind a norm 117 us, 6.0 TB/s; read twice, the second time out of the caches, 126;
  // without a norm, 160 / 300 / 600 / 1,184 rows of 12,288 2.7 / 3.8 / 6.0 / 9.0 us, read twice 4.0 / 4.6 / 6.7 / 10.1, of 16,384 3.2 / 4.9 / 7.3 /
  // 10.7, read twice 5.0 / 6.1 / 8.6 / 12.8), but for float32 behind a norm, which is faster read twice (600 / 8,192 rows of 12,288 24 / 206 us, kept 27 / 302), and for bfloat16 rows without
  // a norm that are not whole, which are where there are many of them or they are long (300 / 1,184 / 8,192 of 12,289 7.1 / 14.1 / 83.6 us, kept
  // 6.0 / 17.3 / 110.8; of 9,001 5.5 / 11.5 / 68.4, kept 3.5 / 9.8 / 61.0).
  if (P.tokens <= sms) {
    if (chunks <= 512) return int8_rows_kept<T, TG, NORM, 1>(P, threads(1), sms, stream);
    if (chunks <= 1024) return int8_rows_kept<T, TG, NORM, 2>(P, threads(2), sms, stream);
    if (chunks <= 512 * INT8_ROW_CHUNKS) return int8_rows_kept<T, TG, NORM, INT8_ROW_CHUNKS>(P, threads(INT8_ROW_CHUNKS), sms, stream);
  } else if (chunks <= 64) {
    // Short rows take a warp each: two warps that meet over a row cost more than the row (8,192 x 512 bfloat16 5.4 -> 3.8 us, behind a
    // norm 8.5 -> 6.3, 8,192 x 64 5.3 -> 2.5).  Up to 128 chunks that holds for bfloat16 (8,192 x 1,024 6.2 -> 5.7, behind a norm
    // 11.1 -> 10.3) where there are many rows (200 x 1,024 behind a norm 2.2 -> 2.5) that are whole, of the others up to 96.
    return P.whole ? int8_rows_warps<T, TG, NORM, 2, true>(P, sms, stream) : int8_rows_warps<T, TG, NORM, 2, false>(P, sms, stream);
  } else if (P.tokens > 4 * sms && chunks <= (P.whole ? sizeof(T) == 2 ? 128 : 0 : 96)) {
    if (!P.whole) return int8_rows_warps<T, TG, NORM, 3, false>(P, sms, stream);
    if constexpr (sizeof(T) == 2) return int8_rows_warps<T, TG, NORM, 4, true>(P, sms, stream);
  } else if (chunks <= 1024) {
    return int8_rows_kept<T, TG, NORM, 2>(P, threads(2), sms, stream);
  } else if constexpr (NORM == (sizeof(T) == 2)) {
    if (chunks <= 2048) return int8_rows_kept<T, TG, NORM, 2, 1024>(P, threads(2), sms, stream);
  } else if constexpr (!NORM) {
    if (chunks <= 2048 && P.whole) return int8_rows_blocks<T, TG, NORM, 2, true, 1024>(P, threads(2), sms, stream);
  }
  return P.whole ? b200_launch(int8_long_rows_kernel<T, TG, NORM, true>, dim3(P.tokens), dim3(512), 0, stream, 0, P)
                                : b200_launch(int8_long_rows_kernel<T, TG, NORM, false>, dim3(P.tokens), dim3(512), 0, stream, 0, P);
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
