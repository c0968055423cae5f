// Log probabilities of given tokens, the entropy and the most likely tokens of float logits [rows, vocab], in one pass.
//
//   m = max l,  s = sum e^(l - m),  w = sum (l - m) e^(l - m)
//   log p(token) = (l_token - m) - log s,   H = log s - w / s,   ties among the most likely go to the lower id.
//
// The bytes of the logits bound it.  Every thread keeps (m, s, w) of its elements in registers and joins them with the
// others' at the end.  The most likely tokens cost the pass nothing but the maximum that it needs anyway: a thread's
// elements form at most CHUNKS chunks, whose maxima stay in registers.  The k-th largest of all chunks' maxima is no
// larger than the k-th largest element, so every one of the k lies in a chunk whose maximum reaches it: as a rule k
// chunks, which are read again (from the second-level cache) and sorted.  That holds for every input: where many
// elements are alike more chunks are read again, up to all, and so they are where less than k of 64 parts hold an element that is not -inf (2,048 rows
// of 151,936 with 20 alternatives 205 us, with 15 ids allowed 1,327; 45 rows 13 and 73).
//
// A row is one CTA's, or, where rows are few, a cluster's: every CTA takes a slice and the first joins what they found
// out of distributed shared memory.
//
// A row with a NaN or +inf, or with -inf alone, has no distribution: its numbers are NaN (a NaN is never among the most
// likely tokens; where less than k tokens are no NaN the missing ids are -1).
#include <cooperative_groups.h>
#include <math.h>

#include "common.cuh"

namespace cg = cooperative_groups;

constexpr int CHUNKS = 8;                 // of a thread; its elements are dealt to them in turn of iterations
constexpr int MOST_TOP = 32;              // a list of the best is a register of a warp's lanes
constexpr int MOST_CLUSTER = 8;
typedef unsigned long long u64;

// Order of floats as whole numbers (no NaN, -0 taken as 0), then the lower id first.
__device__ __forceinline__ u64 key_of(float v, int id) {
  const unsigned bits = __float_as_uint(v + 0.0f);
  const unsigned up = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
  return (static_cast<u64>(up) << 32) | (0xffffffffu - static_cast<unsigned>(id));
}
__device__ __forceinline__ int id_of(u64 key) { return static_cast<int>(0xffffffffu - static_cast<unsigned>(key)); }
__device__ __forceinline__ float value_of(u64 key) {
  const unsigned up = static_cast<unsigned>(key >> 32);
  return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}

// A warp's list: lane i holds the i-th best, best first.
template <typename K>
__device__ __forceinline__ K exchange(K v, int step, bool keep_larger) {
  const K other = __shfl_xor_sync(0xffffffffu, v, step);
  return (other > v) == keep_larger ? other : v;
}
template <typename K>
__device__ __forceinline__ K sort_bitonic(K v) {              // of a bitonic sequence
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int step = 16; step > 0; step >>= 1) v = exchange(v, step, (lane & step) == 0);
  return v;
}
template <typename K>
__device__ __forceinline__ K sort_lanes(K v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int step = size >> 1; step > 0; step >>= 1) v = exchange(v, step, ((lane & step) == 0) == ((lane & size) == 0 || size == 32));
  return v;
}
// The best 32 of two lists (`other`: the other list's entry 31 - lane).
template <typename K>
__device__ __forceinline__ K join_lists(K mine, K other) { return sort_bitonic(other > mine ? other : mine); }
// The lanes' candidates into the list, one after the other; `last`: the list's last entry that counts.
template <typename K>
__device__ __forceinline__ void insert_all(K& list, K mine, bool have, int last) {
  const int lane = threadIdx.x & 31;
  const K least = __shfl_sync(0xffffffffu, list, last);       // (asked by all lanes, whether they have a candidate or not)
  unsigned left = __ballot_sync(0xffffffffu, have && mine > least);
  while (left != 0) {
    const K next = __shfl_sync(0xffffffffu, mine, __ffs(left) - 1);
    left &= left - 1;
    const int place = __popc(__ballot_sync(0xffffffffu, list > next));
    const K up = __shfl_up_sync(0xffffffffu, list, 1);
    list = lane < place ? list : lane == place ? next : up;
  }
}
// The lists of the CTA's first `some` warps joined; all warps hold the result.  `sh`: [WARPS][32].
template <int WARPS, typename K>
__device__ K join_warps(K list, int some, K* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  some = min(some, WARPS);
  for (int half = some > 1 ? 1 << (31 - __clz(some - 1)) : 0; half > 0; half >>= 1) {
    if (warp >= half && warp < 2 * half) sh[warp * 32 + lane] = list;      // (a warp beyond `some` has nothing)
    __syncthreads();
    if (warp < half) list = join_lists(list, sh[(warp + half) * 32 + 31 - lane]);
  }
  if (warp == 0) sh[lane] = list;
  __syncthreads();
  return sh[lane];
}

struct Sums { float m, s, w; };
__device__ __forceinline__ float exp_of(float d) {            // e^d
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(d * 1.4426950408889634f));
  return y;
}
// (a NaN stays one, and -inf becomes a number whose exponential is 0, so that 0 * -inf does not come up)
__device__ __forceinline__ float no_less(float d) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(y) : "f"(d), "f"(-1000.0f));
  return y;
}
// Sums relative to a larger maximum.
__device__ __forceinline__ void raise_to(Sums& a, float m) {
  if (m > a.m) {
    if (a.m > -INFINITY) {
      const float d = a.m - m, f = exp_of(d);
      a.w = f > 0.0f ? f * fmaf(d, a.s, a.w) : 0.0f * a.s;    // (a NaN stays one)
      a.s *= f;
    }
    a.m = m;
  }
}
__device__ __forceinline__ void add_to(Sums& a, Sums b) {
  raise_to(a, b.m);
  raise_to(b, a.m);
  a.s += b.s;
  a.w += b.w;
}
__device__ __forceinline__ void add_element(Sums& a, float v, float base) {
  const float d = no_less(v - base), e = exp_of(d);
  a.s += e;
  a.w = fmaf(e, d, a.w);
}
__device__ __forceinline__ Sums sums_from(const Sums& a, int step) {
  return {__shfl_xor_sync(0xffffffffu, a.m, step), __shfl_xor_sync(0xffffffffu, a.s, step), __shfl_xor_sync(0xffffffffu, a.w, step)};
}

template <int THREADS>
struct Shared {
  static constexpr int WARPS = THREADS / 32;
  float maxima[64];
  u64 keys[WARPS * 32];
  int chunks[CHUNKS * THREADS];           // those whose maximum reaches the k-th largest
  int count;
  Sums sums[WARPS];
  // of the cluster's CTAs, written by each into the first's
  u64 best[MOST_CLUSTER][32];
  Sums parts[MOST_CLUSTER];
};

// grid: rows x cluster.  A row's elements: up to three in front of the first 16-byte boundary, vectors of four, up to three behind.
// UNROLL: 16-byte loads of a thread on their way.
template <int THREADS, int UNROLL, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS)
logprobs_kernel(const float* logits, long long row_stride, int vocab, const int* tokens, int top,
                int cluster, float* __restrict__ logprobs, float* __restrict__ entropy, int* __restrict__ top_ids,
                float* __restrict__ top_logprobs, int* err) {
  constexpr int WARPS = THREADS / 32;
  __shared__ Shared<THREADS> sh;
  const int rank = static_cast<int>(blockIdx.x % cluster);
  const long long row_index = blockIdx.x / cluster;
  const float* row = logits + row_index * row_stride;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  pdl_launch_dependents();
  float given = 0.0f;
  if (rank == 0 && threadIdx.x == 0 && tokens != nullptr) {
    const int token = tokens[row_index];
    if (token < 0 || token >= vocab) {
      atomicOr(err, B200_ERR_TOKEN_RANGE);
      given = NAN;
    } else {
      given = row[token];
    }
  }
  if (threadIdx.x == 0) sh.count = 0;
  if (cluster > 1) cg::this_cluster().barrier_arrive();       // (what is written into the first CTA waits until it has begun)

  const int front = min(vocab, static_cast<int>((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / 4));
  const int vectors = (vocab - front) / 4, behind = front + 4 * vectors;
  const int per = (vectors + cluster - 1) / cluster;
  const int begin = min(vectors, rank * per), end = min(vectors, begin + per);
  const float4* body = reinterpret_cast<const float4*>(row + front);
  const int turns = (end - begin + UNROLL * THREADS - 1) / (UNROLL * THREADS), turns_a_chunk = (turns + CHUNKS - 1) / CHUNKS;

  Sums a = {-INFINITY, 0.0f, 0.0f};
  // the elements outside the vectors: one each of the first CTA's first lanes
  const int loose = front + vocab - behind;
  const int loose_id = static_cast<int>(threadIdx.x) < front ? static_cast<int>(threadIdx.x) : behind + static_cast<int>(threadIdx.x) - front;
  const bool has_loose = rank == 0 && static_cast<int>(threadIdx.x) < loose;
  float loose_value = 0.0f;
  if (has_loose) {
    loose_value = row[loose_id];
    a.m = fmaxf(a.m, loose_value);
    add_element(a, loose_value, a.m == -INFINITY ? 0.0f : a.m);
  }
  float maxima[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    maxima[c] = -INFINITY;
    const int stop = min(turns, (c + 1) * turns_a_chunk);
    for (int t = c * turns_a_chunk; t < stop; ++t) {
      const int at = begin + t * UNROLL * THREADS + static_cast<int>(threadIdx.x);
      float4 v[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        v[u] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (at + u * THREADS < end) v[u] = __ldcg(body + at + u * THREADS);
      }
      float mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) mx = fmaxf(mx, fmaxf(fmaxf(v[u].x, v[u].y), fmaxf(v[u].z, v[u].w)));
      maxima[c] = fmaxf(maxima[c], mx);
      raise_to(a, mx);
      const float base = a.m == -INFINITY ? 0.0f : a.m;
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        add_element(a, v[u].x, base);
        add_element(a, v[u].y, base);
        add_element(a, v[u].z, base);
        add_element(a, v[u].w, base);
      }
    }
  }
#pragma unroll
  for (int step = 16; step > 0; step >>= 1) add_to(a, sums_from(a, step));
  if (lane == 0) sh.sums[warp] = a;

  u64 best = 0;                                               // (0: nothing)
  if (top > 0) {
    // A value that at least `top` chunks reach, and as few others as can be: the top-th largest of 64 parts of the CTA's maxima.
    float mx = maxima[0];
#pragma unroll
    for (int c = 1; c < CHUNKS; ++c) mx = fmaxf(mx, maxima[c]);
    constexpr int PARTS = 64 / WARPS;            // of a warp
#pragma unroll
    for (int step = 16 / PARTS; step > 0; step >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, step));
    if (lane % (32 / PARTS) == 0) sh.maxima[warp * PARTS + lane / (32 / PARTS)] = mx;
    __syncthreads();
    const float list = join_lists(sort_lanes(sh.maxima[lane]), __shfl_xor_sync(0xffffffffu, sort_lanes(sh.maxima[32 + lane]), 31));
    const float reach = __shfl_sync(0xffffffffu, list, top - 1);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
      if (maxima[c] >= reach && c * turns_a_chunk < turns) sh.chunks[atomicAdd(&sh.count, 1)] = c * THREADS + static_cast<int>(threadIdx.x);
    __syncthreads();
    // the chunks' elements (in whatever order they stand there: a list of distinct keys does not depend on it)
    if (warp == 0) insert_all(best, has_loose ? key_of(loose_value, loose_id) : 0ull, has_loose && loose_value == loose_value, top - 1);
    // (all warps share all chunks' elements, AGAIN loads of a lane on their way: one chunk a warp, one load behind the other, were 30 us
    // more for 2,048 rows of 151,936.  In the kernel of few rows few elements are a few warps', whose lists take fewer steps to join: one
    // row with 5 alternatives 8.9 -> 8.7 us, 45 masked rows 9.6 -> 9.4; in that of many 205.3 -> 207.3.)
    constexpr int AGAIN = 4;
    const int elements = turns_a_chunk * UNROLL * 4, all = sh.count * elements;
    const int some = CTAS == 1 && all <= 4 * 32 * AGAIN ? max(1, (all + 32 * AGAIN - 1) / (32 * AGAIN)) : WARPS;
    for (int x0 = warp < some ? warp * 32 : all; x0 < all; x0 += AGAIN * 32 * some) {
      float v[AGAIN];
      int id[AGAIN];
#pragma unroll
      for (int y = 0; y < AGAIN; ++y) {
        const int x = x0 + y * 32 * some + lane;
        id[y] = -1;
        if (x < all) {
          const int i = x / elements, e = x - i * elements, chunk = sh.chunks[i];
          const int turn = chunk / THREADS * turns_a_chunk + e / (UNROLL * 4);
          const int at = begin + turn * UNROLL * THREADS + e / 4 % UNROLL * THREADS + chunk % THREADS;
          if (turn < turns && at < end) id[y] = front + 4 * at + e % 4;
        }
        if (id[y] >= 0) v[y] = __ldcg(row + id[y]);
      }
#pragma unroll
      for (int y = 0; y < AGAIN; ++y) insert_all(best, id[y] >= 0 ? key_of(v[y], id[y]) : 0ull, id[y] >= 0 && v[y] >= reach, top - 1);
    }
    best = join_warps<WARPS>(best, some, sh.keys);
  } else {
    __syncthreads();
  }
  a = sh.sums[lane < WARPS ? lane : 0];
  if (lane >= WARPS) a = {-INFINITY, 0.0f, 0.0f};
#pragma unroll
  for (int step = 16; step > 0; step >>= 1) add_to(a, sums_from(a, step));
  if (cluster > 1) {
    cg::cluster_group all = cg::this_cluster();
    all.barrier_wait();
    if (warp == 0) {
      if (lane == 0) *all.map_shared_rank(&sh.parts[rank], 0) = a;
      *all.map_shared_rank(&sh.best[rank][lane], 0) = best;
    }
    all.sync();
    if (rank != 0) return;
    a = {-INFINITY, 0.0f, 0.0f};
    for (int r = 0; r < cluster; ++r) add_to(a, sh.parts[r]);
    if (top > 0) best = join_warps<WARPS>(warp < cluster ? sh.best[warp][lane] : 0ull, cluster, sh.keys);
  }
  if (warp != 0) return;
  const float log_s = logf(a.s);
  if (lane == 0) {
    if (tokens != nullptr) logprobs[row_index] = (given - a.m) - log_s;
    entropy[row_index] = log_s - a.w / a.s;
  }
  if (lane < top) {
    top_ids[row_index * top + lane] = best != 0 ? id_of(best) : -1;
    top_logprobs[row_index * top + lane] = best != 0 ? (value_of(best) - a.m) - log_s : NAN;
  }
}

// CTAs that share a row: clusters while rows are few, so that all SMs read.  (Clusters of eight find room side by side on half of the
// SMs only: 16 rows of 151,936 with 20 alternatives 16.5 us in eights, where 32 take 11.1 in fours.)
static int cluster_of(int rows, int vocab, int sms) {
  int cluster = 1;
  while (cluster < MOST_CLUSTER && 2 * cluster * rows <= (cluster < 4 ? sms : sms / 2) && vocab / (2 * cluster) >= 4096) cluster *= 2;
  return cluster;
}

// `tokens` (int32 [rows]; with it `logprobs`, float [rows]) may be null; `top_ids` int32 and `top_logprobs` float [rows, top], top <= 32.
B200_EXPORT int b200_token_logprobs(const float* logits, long long row_stride, int rows, int vocab, const int* tokens, int top,
                                    float* logprobs, float* entropy, int* top_ids, float* top_logprobs, int* err,
                                    cudaStream_t stream) {
  if (rows == 0) return 0;
  if (rows < 0 || vocab <= 0 || top < 0 || top > MOST_TOP || top > vocab || row_stride < 0) return B200_BAD_SIZE;
  if (vocab > INT32_MAX - (1 << 20) || rows > INT32_MAX / MOST_CLUSTER) return B200_BAD_SIZE;
  if (logits == nullptr || entropy == nullptr || err == nullptr || (tokens != nullptr && logprobs == nullptr) ||
      (top > 0 && (top_ids == nullptr || top_logprobs == nullptr)))
    return B200_BAD_SIZE;
  int device = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (e != cudaSuccess) return static_cast<int>(e);
  const int cluster = cluster_of(rows, vocab, sms);
  // Few rows: a thread has all of its elements on their way at once where it can.  Many: 1,536 threads an SM, so that some CTAs read
  // while others sort; long rows in CTAs of 512 threads, short ones in 256 (2,048 rows of 151,936 with 20 alternatives: 212 us
  // against 219, of 32,000 with 5: 72 against 63; without alternatives the first take 190, their bytes at the copy rate).
  const bool many = rows >= 2 * sms, small = many && vocab < 65536;
  return b200_launch(small ? logprobs_kernel<256, 4, 6> : many ? logprobs_kernel<512, 4, 3> : logprobs_kernel<512, 10, 1>,
                     dim3(static_cast<unsigned>(rows) * cluster), dim3(small ? 256 : 512), 0, stream, cluster > 1 ? cluster : 0, logits, row_stride, vocab, tokens, top, cluster, logprobs,
                     entropy, top_ids, top_logprobs, err);
}
