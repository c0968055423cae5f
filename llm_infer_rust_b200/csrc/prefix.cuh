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
