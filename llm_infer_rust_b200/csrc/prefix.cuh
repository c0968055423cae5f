// Decode attention of rows that share their first keys: what its kernels have in common.
//
// The rows of a call (one token each) stand in groups.  A group's first `shared` keys are the same for all of its rows and are
// read through the block table of its first row, once for all of them: the group's query vectors of one KV head (rows x query
// heads a KV head) are the rows of one product.  What a row has behind them is its own.  Both parts are cut into splits; every
// split leaves, for each of its query vectors, its maximum m, its sum l = sum 2^(s - m) and its output sum 2^(s - m) v, all in
// float, and one kernel behind them joins a vector's splits.
#pragma once
#include <math.h>

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
  bool shared;
};

// A vector's splits joined, a warp a vector: grid (vectors / MERGE_WARPS), blocks of MERGE_WARPS warps.  The splits' weights
// 2^(m - max) stand in the lanes; a lane owns groups of four dims.  `pitch`: floats of a split's output (a multiple of 4).
constexpr int MERGE_WARPS = 4;
template <typename T, int PITCH>
__global__ void __launch_bounds__(MERGE_WARPS * 32)
prefix_merge_kernel(T* __restrict__ out, const PrefixCall c, int hd) {
  constexpr int MOST = 128;                     // splits in all
  const int lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();
  const long long vec = static_cast<long long>(blockIdx.x) * MERGE_WARPS + (threadIdx.x >> 5);
  if (vec >= static_cast<long long>(c.n_rows) * c.nh) return;
  const int splits = prefix_splits(c);
  const float2* ml = c.part_ml + vec * splits;
  const float* acc = c.part_acc + vec * splits * PITCH;
  float2 mine[MOST / 32];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < MOST / 32; ++k) {
    mine[k] = make_float2(-INFINITY, 0.0f);
    if (k * 32 + lane < splits) mine[k] = ml[k * 32 + lane];
    m = fmaxf(m, mine[k].x);
  }
  m = warp_max(m);
  float l = 0.0f, f[MOST / 32];
#pragma unroll
  for (int k = 0; k < MOST / 32; ++k) {
    f[k] = mine[k].x == -INFINITY ? 0.0f : exp2f(mine[k].x - m);
    l = fmaf(mine[k].y, f[k], l);
  }
  l = warp_sum(l);
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  const int row = static_cast<int>(vec / c.nh), head = static_cast<int>(vec % c.nh);
  T* dst = out + (static_cast<long long>(c.cu_q[c.rows[row]]) * c.nh + head) * hd;
  constexpr int PER = (PITCH + 127) / 128;
  float4 o[PER];
#pragma unroll
  for (int n = 0; n < PER; ++n) o[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int k = 0; k < MOST / 32; ++k) {
    const int some = min(32, splits - 32 * k);
#pragma unroll 4
    for (int s = 0; s < some; ++s) {
      const float w = __shfl_sync(0xffffffffu, f[k], s);
      if (w == 0.0f) continue;                  // (nothing was written where a split saw no key)
      const float* src = acc + static_cast<long long>(32 * k + s) * PITCH;
#pragma unroll
      for (int n = 0; n < PER; ++n) {
        const int dim = n * 128 + lane * 4;
        if (PITCH % 128 == 0 || dim < PITCH) {
          const float4 a = __ldcg(reinterpret_cast<const float4*>(src + dim));
          o[n].x = fmaf(w, a.x, o[n].x);
          o[n].y = fmaf(w, a.y, o[n].y);
          o[n].z = fmaf(w, a.z, o[n].z);
          o[n].w = fmaf(w, a.w, o[n].w);
        }
      }
    }
  }
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    const int dim = n * 128 + lane * 4;
    const float y[4] = {o[n].x * inv, o[n].y * inv, o[n].z * inv, o[n].w * inv};
#pragma unroll
    for (int e = 0; e < 4; e += 2)              // (head sizes are even)
      if (dim + e < hd) {
        dst[dim + e] = from_f32<T>(y[e]);
        dst[dim + e + 1] = from_f32<T>(y[e + 1]);
      }
  }
}
template <typename T, int PITCH>
static inline int prefix_merge(void* out, const PrefixCall& c, int hd, cudaStream_t stream) {
  const long long vectors = static_cast<long long>(c.n_rows) * c.nh;
  return b200_launch(prefix_merge_kernel<T, PITCH>, dim3(static_cast<unsigned>((vectors + MERGE_WARPS - 1) / MERGE_WARPS)), dim3(MERGE_WARPS * 32), 0,
                     stream, 0, static_cast<T*>(out), c, hd);
}
