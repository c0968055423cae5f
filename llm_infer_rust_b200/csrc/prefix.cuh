// Decode attention of rows that share their first keys: what its kernels have in common.
//
// The rows of a call (one token each) stand in groups.  A group's first `shared` keys are the same for all of its rows and are
// read through the block table of its first row, once for all of them: the group's query vectors of one KV head (rows x query
// heads a KV head) are the rows of one product.  What a row has behind them is its own.  Both parts are cut into splits; every
// split leaves, for each of its query vectors, its maximum m, its sum l = sum 2^(s - m) and its output sum 2^(s - m) v, all in
// float, and one kernel behind them joins a vector's splits.
#pragma once
#include <math.h>

#include <initializer_list>

#include "common.cuh"

struct PrefixCall {
  const int* block_table;      // [.., table_stride]
  const int* cu_q;
  const int* kv_len;           // of the batch's rows
  const int* rows;             // [n_rows]: batch rows, group by group
  const int2* groups;          // [n_groups]: (index of its first row in `rows`, shared keys)
  float* part_acc;             // [n_rows * nh][splits][D]
  float2* part_ml;             // [n_rows * nh][splits]
  int* err;
  int table_stride, n_rows, n_groups, nh, nkv, page_size, pages;
  int splits_shared, splits_own;
  int tiles;                   // tiles of a group's vectors that the grid has CTAs for
  float scale_log2;
};

__device__ __forceinline__ int prefix_splits(const PrefixCall& c) { return c.splits_shared + c.splits_own; }

// Asks for the call's index arrays, into the second-level cache, before the kernel may read them (a warp; what is written there after this
// arrives there too): a chain of them, group, row, length, stands in front of the first key.  Of the rows' lengths and tokens the lines that
// they begin in, for which rows there are is not known yet.  (Six groups of 42 rows 28.5 -> 28.2 us, 64 rows behind 32,768 keys 67.9 -> 67.5.)
__device__ __forceinline__ void prefetch_indices(const PrefixCall& c) {
  const int lane = threadIdx.x & 31;
  auto ask = [](const void* p) { asm volatile("prefetch.global.L2 [%0];\n" ::"l"(p)); };
  if (lane * 8 < c.n_rows) ask(c.rows + lane * 8);
  if (lane * 4 < c.n_groups) ask(c.groups + lane * 4);
  if (lane < 8) ask(reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(lane < 4 ? c.kv_len : c.cu_q) & ~uintptr_t(127)) + (lane & 3) * 32);
}

// (first row, rows) of group g, inside the call's rows whatever the array says.
__device__ __forceinline__ int2 rows_of_group(const PrefixCall& c, int g) {
  const int first = min(max(c.groups[g].x, 0), c.n_rows);
  const int end = g + 1 < c.n_groups ? min(max(c.groups[g + 1].x, first), c.n_rows) : c.n_rows;
  return make_int2(first, end - first);
}

// Keys of batch row `row`, no more than its block table has places for.
__device__ __forceinline__ int keys_of_row(const PrefixCall& c, int row) {
  const int keys = max(c.kv_len[row], 0);
  const long long most = static_cast<long long>(c.table_stride) * c.page_size;
  if (keys <= most) return keys;
  atomicOr(c.err, B200_ERR_SLOT_RANGE);
  return static_cast<int>(most);
}
__device__ __forceinline__ int shared_of_group(const PrefixCall& c, int g) {
  const int keys = max(c.groups[g].y, 0);
  const long long most = static_cast<long long>(c.table_stride) * c.page_size;
  if (keys <= most) return keys;
  atomicOr(c.err, B200_ERR_SLOT_RANGE);
  return static_cast<int>(most);
}

// The group of the i-th row: the last one that begins at or before it (a whole warp asks).
__device__ __forceinline__ int group_of_row(const PrefixCall& c, int i) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int g0 = 0; g0 < c.n_groups; g0 += 32) {
    const bool begun = g0 + lane < c.n_groups && c.groups[g0 + lane].x <= i;
    const unsigned which = __ballot_sync(0xffffffffu, begun);
    before += __popc(which);
    if (which != 0xffffffffu) break;
  }
  return before - 1;
}

// Whether a call's operands are there, and its keys, blocks and splits can be counted in 32 bits.
static inline bool prefix_can_be_served(std::initializer_list<const void*> operands, const int* groups, int n_groups, int table_stride, int page_size) {
  for (const void* p : operands)
    if (p == nullptr) return false;
  return (groups != nullptr || n_groups == 0) && static_cast<long long>(table_stride) * page_size <= (1 << 30);
}

// Sets a kernel's limit of shared memory, once a device (`seen`: the kernel's own, one for each of the first 16 devices).
template <typename Kernel>
static inline int prefix_smem_limit(Kernel kernel, int bytes, bool (&seen)[16]) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && (device >= 16 || !seen[device])) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && device < 16) seen[device] = true;
  }
  return static_cast<int>(e);
}

// What a CTA works on: `vectors` query vectors of one KV head, keys [begin, end) of one block table.
struct PrefixItem {
  const int* table;
  int i0, vector0, vectors;    // vector v: row i0 + (vector0 + v) / group of `rows`, query head kvh * group + (vector0 + v) % group
  int begin, end, kvh, slot;
};

// A part's maximum and sum as they are stored.  Scores that are all NaN leave no maximum; the sum, NaN too, must not be taken for that of a
// part without keys.
__device__ __forceinline__ float2 part_of(float m, float l) { return make_float2(l != l && m == -INFINITY ? 0.0f : m, l); }

__device__ __forceinline__ float prefix_exp2(float x) {      // 2^x, one special-function instruction (-inf gives 0)
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// One vector out of its `count` parts, rows of PITCH floats of which `hd` are the head's: the CTA's warps share the parts, up to BATCH of them a
// turn, maxima and sums asked for together with the outputs that they weight, for what this takes is a few answers from the
// second-level cache one behind the other.  `where`: the place of part p's maximum and sum, and of its outputs.  `left`: shared memory.
// CHECKED: false, and nothing written, where an output or a sum is no number or an infinity, or an output is below 2^-80 and not zero (the
// largest weight behind each is 1).
template <int PITCH, int WARPS>
struct JoinShared { float row[WARPS][PITCH + 4]; };
template <int PITCH, int WARPS, bool CHECKED = false, typename T, typename Where>
__device__ __forceinline__ bool join_parts(T* __restrict__ dst, int hd, int count, const Where& where, JoinShared<PITCH, WARPS>& left) {
  constexpr int PER = (PITCH + 127) / 128, BATCH = PER == 1 ? 8 : PER == 2 ? 4 : 2;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float4 o[PER];
#pragma unroll
  for (int n = 0; n < PER; ++n) o[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float m = -INFINITY, l = 0.0f;
  for (int p0 = warp * BATCH; p0 < count; p0 += WARPS * BATCH) {
    float4 a[BATCH][PER];
    float2 ml[BATCH];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const float2* of_part;
      const float* src;
      where(min(p0 + b, count - 1), of_part, src);
      ml[b] = __ldcg(of_part);
#pragma unroll
      for (int n = 0; n < PER; ++n)
        if (PITCH % 128 == 0 || n * 128 + lane * 4 < PITCH) a[b][n] = __ldcg(reinterpret_cast<const float4*>(src + n * 128 + lane * 4));
    }
    float most = m;
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      if (p0 + b >= count) ml[b] = make_float2(-INFINITY, 0.0f);
      most = fmaxf(most, ml[b].x);
    }
    if (most == -INFINITY) continue;
    const float f = prefix_exp2(m - most);         // (0 on the first visible part)
    m = most;
    l *= f;
#pragma unroll
    for (int n = 0; n < PER; ++n) { o[n].x *= f; o[n].y *= f; o[n].z *= f; o[n].w *= f; }
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      if (ml[b].x == -INFINITY) continue;          // (where a split saw no key nothing was written)
      const float w = prefix_exp2(ml[b].x - m);
      l = fmaf(ml[b].y, w, l);
#pragma unroll
      for (int n = 0; n < PER; ++n) {
        o[n].x = fmaf(w, a[b][n].x, o[n].x);
        o[n].y = fmaf(w, a[b][n].y, o[n].y);
        o[n].z = fmaf(w, a[b][n].z, o[n].z);
        o[n].w = fmaf(w, a[b][n].w, o[n].w);
      }
    }
  }
  // the warps' parts: columns are the threads' from here on (some have none)
#pragma unroll
  for (int n = 0; n < PER; ++n)
    if (PITCH % 128 == 0 || n * 128 + lane * 4 < PITCH) *reinterpret_cast<float4*>(left.row[warp] + n * 128 + lane * 4) = o[n];
  if (lane == 0) { left.row[warp][PITCH] = m; left.row[warp][PITCH + 1] = l; }
  if constexpr (CHECKED) {
    bool settled = fabsf(l) < INFINITY;
    const auto look = [&](float x) { settled = settled && fabsf(x) < INFINITY && (fabsf(x) >= 8.2718061e-25f || x == 0.0f); };
#pragma unroll
    for (int n = 0; n < PER; ++n)
      if (PITCH % 128 == 0 || n * 128 + lane * 4 < PITCH) { look(o[n].x); look(o[n].y); look(o[n].z); look(o[n].w); }
    if (__syncthreads_or(!settled)) return false;
  } else {
    __syncthreads();
  }
  const int warps = min(WARPS, (count + BATCH - 1) / BATCH);      // that had parts
  float most = -INFINITY, sum = 0.0f;
  for (int w = 0; w < warps; ++w) most = fmaxf(most, left.row[w][PITCH]);
  const float base = most == -INFINITY ? 0.0f : most;
  for (int w = 0; w < warps; ++w) sum = fmaf(left.row[w][PITCH + 1], prefix_exp2(left.row[w][PITCH] - base), sum);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;             // (a row of no keys gets zeros, a NaN stays one)
  for (int dim = 2 * static_cast<int>(threadIdx.x); dim < hd; dim += 2 * WARPS * 32) {      // (head sizes are even)
    float x = 0.0f, y = 0.0f;
    for (int w = 0; w < warps; ++w) {
      const float2 two = *reinterpret_cast<const float2*>(left.row[w] + dim);
      const float f = prefix_exp2(left.row[w][PITCH] - base);
      x = fmaf(two.x, f, x);
      y = fmaf(two.y, f, y);
    }
    dst[dim] = from_f32<T>(x * inv);
    dst[dim + 1] = from_f32<T>(y * inv);
  }
  return true;
}
// Warps of a CTA that joins one of `vectors` vectors.  Few vectors have many parts each, a hundred and more where one prompt's keys are all there
// is: then all of them at once, while an SM has a CTA.  Many have a dozen, and all vectors are to be on the SMs at once.  (4 / 16 warps: two
// rows of 16 heads behind 4,096 keys 18.6 / 13.4 us in all, 32 rows behind 512 keys 15.0 / 19.0; 2 / 4 warps: 768 vectors 22.6 / 22.0, 1,536
// 27.2 / 27.5, 2,048 65.2 / 67.8 and 92.7 / 96.4.)
static inline int join_warps_of(long long vectors, int sms) { return vectors <= sms ? 16 : vectors <= 2 * sms ? 8 : vectors <= 10 * sms ? 4 : 2; }
