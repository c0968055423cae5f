// Tensor-core attention over the paged bfloat16 cache, for one head size
// (compile with -DHEAD_DIM=<multiple of 16, at most 256>).
//
// Decode (one query position per row) is bound by the bytes of keys and values
// that a step has to read, so this kernel is built around the copy engine.  The
// cache is laid out [page][KV head][offset in page][head_dim]: the rows of one
// page and KV head are one contiguous block, which TMA fetches as boxes of
// (up to 32 rows) x (64 dims = 128 bytes) straight into shared memory in the
// 128-byte swizzle, reporting to an mbarrier.  A CTA owns one (row, KV head,
// split of the keys); each of its warps walks its own blocks of 32 keys through a
// private ring of stages (16 KB per block at head size 128), so that tens of KB
// per SM are in flight and the loop has no block-wide barrier.  Every wait on a
// barrier is bounded by the clock: when it runs out the kernel flags the engine's
// error word, gives the outstanding copies a bounded time to land and returns.
// The arithmetic rides on mma.sync m16n8k16 (bfloat16 in, float accumulate): the
// query heads that share the KV head are the 16 rows of the A operand (at most 16
// heads per KV head; larger groups, page sizes that are no power of two and float
// caches take the CUDA-core kernel of attention.cu), keys and values are read
// from the swizzled tiles with ldmatrix (values transposed).  Scores, the running
// maximum, the running sum and the output are float; probabilities are rounded to
// bfloat16 only as the A operand of P.V, as the values themselves are bfloat16.
//
// Semantics are those of attention.cu (reference: src/models/attention/backend.rs:1455-1498):
// KV head = head / group, score = q.k * scale, keys j <= p (and j > p - W with a
// window), softmax in float, output = P.V.  Value rows at or beyond the sequence
// end are zeroed in shared memory before they are used, key rows there are masked:
// a page that is used again may hold anything.
#include <cooperative_groups.h>

#include "attention_mma.cuh"
#include "kv_map.cuh"

namespace cg = cooperative_groups;

// ------------------------------------------------------------------ decoded tokens
// grid (splits, nkv, decode rows).  Partials: part_acc[((row * nh + head) * splits + split) * D + dim]
// (unnormalised), part_ml[...][2] = (maximum in log2 units, sum).
// Shared memory: [WARPS][STAGES] tiles (1024-byte aligned), the query tile [16][LD], the barriers.
// CTAs start in the grid's order, so the caller lists the rows with the most keys first: in a grid of several waves the short
// ones then fill the gaps behind them (45 rows of 100 to 2,000 keys x 8 KV heads, four query heads each: 45.9 us in the batch's
// order, 41.3 by length).  Ranked by every CTA for itself the same rows took 42.5 us, and rows of one length paid for nothing
// (64 of 512 keys, two query heads: 33.7 -> 35.1 us; 128 of 1,000: 101.6 -> 109.3).
template <int WARPS, int STAGES, bool SHAPED>
__global__ void __launch_bounds__(WARPS * 32, 1)
decode_mma_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                  const bf16* __restrict__ q, bf16* __restrict__ out, float* __restrict__ part_acc,
                  float* __restrict__ part_ml, const int* __restrict__ block_table, int table_stride,
                  const int* __restrict__ cu_q, const int* __restrict__ kv_len, const int* __restrict__ rows, int nh,
                  int nkv, int page_size, int box_rows, int window, ScoreForm sf, int cluster_merge, int* err) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  bf16* qs = reinterpret_cast<bf16*>(tiles + static_cast<size_t>(WARPS) * STAGES * TILE_BYTES);   // [16][LD]
  uint64_t* bars = reinterpret_cast<uint64_t*>(qs + QROWS * LD);                                   // [WARPS][STAGES]

  pdl_launch_dependents();
  if (threadIdx.x < WARPS * STAGES) mbar_init(bars + threadIdx.x, 1);
  asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  __syncthreads();
  // The kernel before this one in the stream wrote q and the step's newest key and value of every row.  The
  // step's index arrays were uploaded before the step's first kernel, and all other keys and values are older:
  // both may be read while that kernel still runs.
  const int splits = gridDim.x, split = blockIdx.x, kvh = blockIdx.y;
  const int row = rows[blockIdx.z];
  const int group = nh / nkv, head0 = kvh * group;
  const int tok = cu_q[row];
  const int kv_end = kv_len[row];
  const int qp = kv_end - 1;
  int k_begin = window > 0 ? max(0, qp - window + 1) : 0;
  if (sf.chunk > 0) k_begin = max(k_begin, qp - qp % sf.chunk);
  k_begin -= k_begin % KB;
  const int blocks_total = (kv_end - k_begin + KB - 1) / KB;
  const int per_split = (blocks_total + splits - 1) / splits;
  const int blk_lo = split * per_split, blk_hi = min(blocks_total, blk_lo + per_split);
  const int* table = block_table + static_cast<size_t>(row) * table_stride;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  unsigned char* my = tiles + static_cast<size_t>(warp) * STAGES * TILE_BYTES;
  uint64_t* my_bars = bars + warp * STAGES;
  int issue = blk_lo + warp;
  int page = 0;
  auto first_fill = [&]() {                            // the ring's first STAGES - 1 blocks of this warp
    page = issue < blk_hi ? lane_page(table, page_size, box_rows, k_begin + issue * KB, kv_end, lane) : 0;
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
      const int next = issue + WARPS;
      const int next_page = next < blk_hi ? lane_page(table, page_size, box_rows, k_begin + next * KB, kv_end, lane) : 0;
      if (issue < blk_hi)
        fetch_block(my + s * TILE_BYTES, &kmap, &vmap, page, page_size, nkv, kvh, box_rows, k_begin + issue * KB, kv_end,
                    my_bars + s, lane);
      issue = next;
      page = next_page;
    }
  };
  // They are fetched under the tail of the kernel before, unless the newest key (position kv_end - 1) is in them.
  const int last_of_fill = blk_lo + warp + (STAGES - 2) * WARPS;
  const bool early = k_begin + (last_of_fill + 1) * KB <= qp;
  if (early) first_fill();
  pdl_wait();
  if (!early) first_fill();

  for (int c = threadIdx.x; c < QROWS * (D / 8); c += blockDim.x) {
    const int r = c / (D / 8), part = c - r * (D / 8);
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (r < group) v = *reinterpret_cast<const uint4*>(q + (static_cast<size_t>(tok) * nh + head0 + r) * D + part * 8);
    *reinterpret_cast<uint4*>(qs + r * LD + part * 8) = v;
  }
  __syncthreads();
  const int g = lane >> 2;
  const int qpos0 = g < group ? qp : -1, qpos1 = g + 8 < group ? qp : -1;
  WarpAcc st;
  st.init();
  int stage = 0;
  uint32_t parity = 0;
  for (int blk = blk_lo + warp; blk < blk_hi; blk += WARPS) {
    const int s_issue = stage == 0 ? STAGES - 1 : stage - 1;      // the stage that the previous block left
    const int next = issue + WARPS;
    const int next_page = next < blk_hi ? lane_page(table, page_size, box_rows, k_begin + next * KB, kv_end, lane) : 0;
    if (issue < blk_hi)
      fetch_block(my + s_issue * TILE_BYTES, &kmap, &vmap, page, page_size, nkv, kvh, box_rows, k_begin + issue * KB,
                  kv_end, my_bars + s_issue, lane);
    issue = next;
    page = next_page;
    if (!mbar_wait(my_bars + stage, parity, err)) {
      // Give the copies that are still in flight a bounded time to land before the tiles are reused.
      for (int s = 0; s < STAGES; ++s) mbar_wait(my_bars + s, s < stage ? parity ^ 1u : parity, err);
      break;
    }
    unsigned char* t = my + stage * TILE_BYTES;
    const int first_key = k_begin + blk * KB;
    if (first_key + KB > kv_end && first_key + lane >= kv_end) {
      // Value rows beyond the sequence: whatever the page holds there must not reach P.V.
      const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int c = 0; c < VALUE_CHUNKS; ++c) *reinterpret_cast<uint4*>(t + V_OFFSET + (c >> 3) * HALF_BYTES + lane * 128 + (c & 7) * 16) = zero;
    }
    __syncwarp();
    if (first_key + KB <= kv_end && (window <= 0 || first_key > qp - window) &&
        (sf.chunk <= 0 || first_key >= qp - qp % sf.chunk))
      block_mma<false, SHAPED>(qs, t, t + V_OFFSET, first_key, kv_end, window, qpos0, qpos1, sf, st);
    else
      block_mma<true, SHAPED>(qs, t, t + V_OFFSET, first_key, kv_end, window, qpos0, qpos1, sf, st);
    __syncwarp();                                      // every lane is done reading before the stage is refilled
    if (++stage == STAGES) { stage = 0; parity ^= 1u; }
  }
  st.l[0] += __shfl_xor_sync(0xffffffffu, st.l[0], 1); st.l[0] += __shfl_xor_sync(0xffffffffu, st.l[0], 2);
  st.l[1] += __shfl_xor_sync(0xffffffffu, st.l[1], 1); st.l[1] += __shfl_xor_sync(0xffffffffu, st.l[1], 2);
  __syncthreads();
  // Merge the warps through shared memory: [WARPS][group][D + 2] floats over the tile area.
  float* merge = reinterpret_cast<float*>(tiles);     // all copies have landed and been used
  constexpr int MS = DV + 2;
  const int ow = kShared ? sf.out_width : DV, oc = kShared ? sf.out_col0 : 0;     // an output row and this launch's columns
  float* mine = merge + WARPS * QROWS * MS;           // [group][MS]: the CTA's own combined part
  // DIFF: the pairs of finished outputs [group][MS] in shared memory become the stored heads, a warp a head
  auto store_differences = [&](const float* done) {
    __syncthreads();
    for (int j = warp; j < group / 2; j += WARPS) {
      const float* a = done + 2 * j * MS;
      const float* b = a + MS;
      float ss = 0.0f;
      for (int dim = lane; dim < DV; dim += 32) {
        const float o = fmaf(-sf.diff_lambda, b[dim], a[dim]);
        ss = fmaf(o, o, ss);
      }
      const float f = sf.diff_gain / sqrtf(warp_sum(ss) / static_cast<float>(DV) + sf.diff_eps);
      bf16* dst = out + (static_cast<size_t>(tok) * (nh / 2) + head0 / 2 + j) * DV;
      for (int dim = lane; dim < DV; dim += 32) dst[dim] = __float2bfloat16_rn(fmaf(-sf.diff_lambda, b[dim], a[dim]) * f);
    }
  };
  const int t2 = (lane & 3) * 2;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = g + 8 * half;
    if (r < group) {
      float* dst = merge + (warp * group + r) * MS;
#pragma unroll
      for (int dn = 0; dn < DV / 8; ++dn) {
        dst[dn * 8 + t2] = st.o[dn][2 * half];
        dst[dn * 8 + t2 + 1] = st.o[dn][2 * half + 1];
      }
      if ((lane & 3) == 0) { dst[DV] = st.m[half]; dst[DV + 1] = st.l[half]; }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < group * DV; i += blockDim.x) {
    const int r = i / DV, dim = i - r * DV;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, merge[(w * group + r) * MS + DV]);
    float l = 0.0f, o = 0.0f;
    if (m != -INFINITY) {
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float* src = merge + (w * group + r) * MS;
        const float f = exp2f(src[DV] - m);
        l += src[DV + 1] * f;
        o += src[dim] * f;
      }
    }
    const int head = head0 + r;
    if (splits == 1) {
      l = with_sink(sf, head, m, l);
      const float y = l > 0.0f ? o / l : 0.0f;
      if constexpr (kDiff) mine[r * MS + dim] = y;
      else out[(static_cast<size_t>(tok) * nh + head) * ow + oc + dim] = __float2bfloat16_rn(y);
    } else if (cluster_merge) {
      mine[r * MS + dim] = o;                          // this CTA's part, for the cluster's first CTA to read
      if (dim == 0) { mine[r * MS + DV] = m; mine[r * MS + DV + 1] = l; }
    } else {
      const size_t slot = (static_cast<size_t>(blockIdx.z) * nh + head) * splits + split;
      part_acc[slot * DV + dim] = o;
      if (dim == 0) { part_ml[slot * 2] = m; part_ml[slot * 2 + 1] = l; }
    }
  }
  if constexpr (kDiff) {
    if (splits == 1) store_differences(mine);
  }
  if (!cluster_merge) return;
  // The splits of a (row, KV head) pair are the CTAs of one cluster: the first combines all parts out of the others'
  // shared memory (every CTA reaches both barriers, also one whose waits ran out).
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  if (split == 0) {
    for (int i = threadIdx.x; i < group * DV; i += blockDim.x) {
      const int r = i / DV, dim = i - r * DV;
      float m = -INFINITY;
      for (int s = 0; s < splits; ++s) m = fmaxf(m, cluster.map_shared_rank(mine, s)[r * MS + DV]);
      float l = 0.0f, o = 0.0f;
      if (m != -INFINITY) {
        for (int s = 0; s < splits; ++s) {
          const float* src = cluster.map_shared_rank(mine, s) + r * MS;
          const float f = exp2f(src[DV] - m);
          l += src[DV + 1] * f;
          o += src[dim] * f;
        }
        l = with_sink(sf, head0 + r, m, l);
      }
      const float y = l > 0.0f ? o / l : 0.0f;
      if constexpr (kDiff) merge[r * MS + dim] = y;      // (the warps' parts there have been used)
      else out[(static_cast<size_t>(tok) * nh + head0 + r) * ow + oc + dim] = __float2bfloat16_rn(y);
    }
    if constexpr (kDiff) store_differences(merge);
  }
  cluster.sync();                                      // nobody leaves while its shared memory may still be read
}

// DIFF.  grid (decode rows, nh / 2): combines the splits of a head's two maps and stores their difference.
__global__ void decode_mma_merge_diff_kernel(bf16* __restrict__ out, const float* __restrict__ part_acc,
                                             const float* __restrict__ part_ml, const int* __restrict__ cu_q,
                                             const int* __restrict__ rows, int nh, int splits, float lambda, float gain,
                                             float eps) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float scratch[33];
  constexpr int PER = (DV + 63) / 64;                   // columns of a thread (the launcher gives at least 64 threads)
  const int tok = cu_q[rows[blockIdx.x]];
  float y[PER] = {};
  for (int map = 0; map < 2; ++map) {
    const size_t base = (static_cast<size_t>(blockIdx.x) * nh + 2 * blockIdx.y + map) * splits;
    float m = -INFINITY;
    for (int s = 0; s < splits; ++s) m = fmaxf(m, part_ml[(base + s) * 2]);
    if (m == -INFINITY) continue;
    float l = 0.0f, o[PER] = {};
    for (int s = 0; s < splits; ++s) {
      const float f = exp2f(part_ml[(base + s) * 2] - m);
      l += part_ml[(base + s) * 2 + 1] * f;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int dim = threadIdx.x + i * blockDim.x;
        if (dim < DV) o[i] += part_acc[(base + s) * DV + dim] * f;
      }
    }
    const float w = (map == 0 ? 1.0f : -lambda) / l;
#pragma unroll
    for (int i = 0; i < PER; ++i) y[i] = fmaf(w, o[i], y[i]);
  }
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < PER; ++i) ss = fmaf(y[i], y[i], ss);
  const float f = gain / sqrtf(block_sum(ss, scratch) / static_cast<float>(DV) + eps);
  bf16* dst = out + (static_cast<size_t>(tok) * (nh / 2) + blockIdx.y) * DV;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int dim = threadIdx.x + i * blockDim.x;
    if (dim < DV) dst[dim] = __float2bfloat16_rn(y[i] * f);
  }
}

// grid (decode rows, nh): combines the splits of one head (maxima are in log2 units).
__global__ void decode_mma_merge_kernel(bf16* __restrict__ out, const float* __restrict__ part_acc,
                                        const float* __restrict__ part_ml, const int* __restrict__ cu_q,
                                        const int* __restrict__ rows, int nh, int splits,
                                        const float* __restrict__ sinks, int out_width, int out_col0) {
  pdl_launch_dependents();
  pdl_wait();
  const int head = blockIdx.y;
  const int tok = cu_q[rows[blockIdx.x]];
  const size_t base = (static_cast<size_t>(blockIdx.x) * nh + head) * splits;
  float m = -INFINITY;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, part_ml[(base + s) * 2]);
  for (int dim = threadIdx.x; dim < DV; dim += blockDim.x) {
    float l = 0.0f, o = 0.0f;
    if (m != -INFINITY) {
      for (int s = 0; s < splits; ++s) {
        const float f = exp2f(part_ml[(base + s) * 2] - m);
        l += part_ml[(base + s) * 2 + 1] * f;
        o += part_acc[(base + s) * DV + dim] * f;
      }
      if (sinks != nullptr && l > 0.0f) l += exp2f(sinks[head] * 1.4426950408889634f - m);
    }
    out[(static_cast<size_t>(tok) * nh + head) * out_width + out_col0 + dim] = __float2bfloat16_rn(l > 0.0f ? o / l : 0.0f);
  }
}

// ------------------------------------------------------------------ prompt portions
// grid (query tiles, nkv, prefill rows).  A CTA serves PF_WARPS * 16 query vectors: consecutive
// tokens of one row x the `group` query heads of one KV head; warp w owns vectors 16 w .. 16 w + 15
// (a warp holds 16 / group whole tokens).  All warps read the same key blocks, which one warp fetches
// into a ring of stages: full[s] flips when the boxes of a block have landed, empty[s] when every
// warp has finished with it.  Each query vector has its own position, so the causal mask (and the
// window) is applied per row of the score tile.
constexpr int PF_WARPS = 4;
// Three CTAs share an SM for heads up to 128 wide (the register budget that this leaves is 170 a thread).
constexpr int PF_MIN_CTAS = D <= 128 && DV <= 128 ? 3 : 1;
constexpr int PF_ROWS = PF_WARPS * 16;

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}

template <int STAGES, bool SHAPED>
__global__ void __launch_bounds__(PF_WARPS * 32, PF_MIN_CTAS)
prefill_mma_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                   const bf16* __restrict__ q, bf16* __restrict__ out, const int* __restrict__ block_table,
                   int table_stride, const int* __restrict__ cu_q, const int* __restrict__ kv_len,
                   const int* __restrict__ prefix_len, const int* __restrict__ rows, int nh, int nkv, int page_size,
                   int box_rows, int window, ScoreForm sf, int* err) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  bf16* qs = reinterpret_cast<bf16*>(tiles + static_cast<size_t>(STAGES) * TILE_BYTES);     // [PF_ROWS][LD]
  uint64_t* full = reinterpret_cast<uint64_t*>(qs + PF_ROWS * LD);
  uint64_t* empty = full + STAGES;

  // Grid: x = KV head, y = row, z = tile order.  CTAs start in the order x, y, z, and a row's last tiles see the
  // most keys: every row's heaviest tiles start first, over all heads, so that the short ones fill the tail.
  const int row = rows[blockIdx.y];
  const int kvh = blockIdx.x;
  const int group = nh / nkv, head0 = kvh * group;
  const int tokens_per_warp = 16 / group;                       // whole tokens per warp
  const int tile_tokens = tokens_per_warp * PF_WARPS;
  const int q_begin = cu_q[row], q_len = cu_q[row + 1] - q_begin;
  const int tile = (q_len + tile_tokens - 1) / tile_tokens - 1 - static_cast<int>(blockIdx.z);
  if (tile < 0) return;
  const int tok0 = tile * tile_tokens;
  const int ntok = min(tile_tokens, q_len - tok0);
  const int prefix = prefix_len[row];
  const int kv_end = min(kv_len[row], prefix + tok0 + ntok);     // causal: nothing later is visible to this tile
  const int p_lo = prefix + tok0;
  int k_begin = window > 0 ? max(0, p_lo - window + 1) : 0;
  if (sf.chunk > 0) k_begin = max(k_begin, p_lo - p_lo % sf.chunk);
  k_begin -= k_begin % KB;
  const int nblk = (kv_end - k_begin + KB - 1) / KB;
  const int* table = block_table + static_cast<size_t>(row) * table_stride;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  for (int c = threadIdx.x; c < PF_ROWS * (D / 8); c += blockDim.x) {
    const int r = c / (D / 8), part = c - r * (D / 8);
    const int w = r >> 4, i = r & 15;
    const int tok = w * tokens_per_warp + i / group, head = head0 + i % group;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (i < tokens_per_warp * group && tok < ntok)
      v = *reinterpret_cast<const uint4*>(q + (static_cast<size_t>(q_begin + tok0 + tok) * nh + head) * D + part * 8);
    *reinterpret_cast<uint4*>(qs + r * LD + part * 8) = v;
  }
  if (threadIdx.x < STAGES) { mbar_init(full + threadIdx.x, 1); mbar_init(empty + threadIdx.x, PF_WARPS); }
  asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  __syncthreads();

  // Positions of this thread's two score rows (lane / 4 and lane / 4 + 8 of the warp's 16 vectors).
  const int g = lane >> 2;
  int qpos[2], tok_of[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = g + 8 * h;
    const int tok = warp * tokens_per_warp + i / group;
    const bool used = i < tokens_per_warp * group && tok < ntok;
    tok_of[h] = used ? tok : -1;
    qpos[h] = used ? p_lo + tok : -1;
  }
  // The warp's own range of key blocks: from its first visible key to its last query's position.
  const int w_tok_lo = warp * tokens_per_warp;
  const int w_tok_hi = min(ntok, w_tok_lo + tokens_per_warp) - 1;           // < w_tok_lo: the warp holds no token
  const int w_p_hi = p_lo + w_tok_hi;
  int w_first_key = window > 0 ? max(0, p_lo + w_tok_lo - window + 1) : 0;
  if (sf.chunk > 0) w_first_key = max(w_first_key, (p_lo + w_tok_lo) - (p_lo + w_tok_lo) % sf.chunk);

  WarpAcc st;
  st.init();
  const bf16* my_q = qs + warp * 16 * LD;
  bool ok = true;
  int page = 0;
  if (warp == 0) {                                                          // prologue of the producer
    page = nblk > 0 ? lane_page(table, page_size, box_rows, k_begin, kv_end, lane) : 0;
    for (int j = 0; j < STAGES - 1 && j < nblk; ++j) {
      const int next_page = j + 1 < nblk ? lane_page(table, page_size, box_rows, k_begin + (j + 1) * KB, kv_end, lane) : 0;
      fetch_block(tiles + j * TILE_BYTES, &kmap, &vmap, page, page_size, nkv, kvh, box_rows, k_begin + j * KB, kv_end,
                  full + j, lane);
      page = next_page;
    }
  }
  for (int it = 0; it < nblk && ok; ++it) {
    const int s = it % STAGES;
    if (warp == 0) {
      const int j = it + STAGES - 1;
      if (j < nblk) {
        const int sj = j % STAGES, use = j / STAGES;
        const int next_page = j + 1 < nblk ? lane_page(table, page_size, box_rows, k_begin + (j + 1) * KB, kv_end, lane) : 0;
        if (use > 0) ok = mbar_wait(empty + sj, (use - 1) & 1, err);          // every warp has left block j - STAGES
        if (ok)
          fetch_block(tiles + sj * TILE_BYTES, &kmap, &vmap, page, page_size, nkv, kvh, box_rows, k_begin + j * KB,
                      kv_end, full + sj, lane);
        page = next_page;
      }
    }
    ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
    if (!ok) break;
    if (!mbar_wait(full + s, (it / STAGES) & 1, err)) { ok = false; break; }
    unsigned char* t = tiles + s * TILE_BYTES;
    const int first_key = k_begin + it * KB;
    if (first_key + KB > kv_end && first_key + lane >= kv_end) {
      // Value rows beyond what this tile may see hold whatever the page or the stage held before (they are
      // masked for every query of the tile): keep them out of P.V.
      const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int c = 0; c < VALUE_CHUNKS; ++c) *reinterpret_cast<uint4*>(t + V_OFFSET + (c >> 3) * HALF_BYTES + lane * 128 + (c & 7) * 16) = zero;
    }
    __syncwarp();
    if (w_tok_hi >= w_tok_lo && first_key <= w_p_hi && first_key + KB > w_first_key) {
      // All keys of the block lie at or before the warp's first query (and inside its last query's window)?
      const bool all_visible = first_key + KB - 1 <= p_lo + w_tok_lo && first_key + KB <= kv_end &&
                               (window <= 0 || first_key > w_p_hi - window) &&
                               (sf.chunk <= 0 || first_key >= w_p_hi - w_p_hi % sf.chunk);
      if (all_visible)
        block_mma<false, SHAPED>(my_q, t, t + V_OFFSET, first_key, kv_end, window, qpos[0], qpos[1], sf, st);
      else
        block_mma<true, SHAPED>(my_q, t, t + V_OFFSET, first_key, kv_end, window, qpos[0], qpos[1], sf, st);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + s);
  }
  if (!ok) {
    // A wait ran out: let the copies in flight land (bounded) before the CTA gives up its shared memory.
    for (int s = 0; s < STAGES; ++s) { mbar_wait(full + s, 0, err); }
    return;
  }
  st.l[0] += __shfl_xor_sync(0xffffffffu, st.l[0], 1); st.l[0] += __shfl_xor_sync(0xffffffffu, st.l[0], 2);
  st.l[1] += __shfl_xor_sync(0xffffffffu, st.l[1], 1); st.l[1] += __shfl_xor_sync(0xffffffffu, st.l[1], 2);
  const int t2 = (lane & 3) * 2;
  if constexpr (kDiff) {
    // a head's two maps are neighbouring rows of the tile: rows g and g ^ 1, that is lanes 4 apart
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float inv = st.l[h] > 0.0f ? 1.0f / st.l[h] : 0.0f;
      const float w = (g & 1) ? -sf.diff_lambda * inv : inv;
      float ss = 0.0f;
#pragma unroll
      for (int dn = 0; dn < DV / 8; ++dn) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float mine = st.o[dn][2 * h + e] * w;
          const float o = mine + __shfl_xor_sync(0xffffffffu, mine, 4);
          st.o[dn][2 * h + e] = o;
          ss = fmaf(o, o, ss);
        }
      }
      ss += __shfl_xor_sync(0xffffffffu, ss, 1);
      ss += __shfl_xor_sync(0xffffffffu, ss, 2);
      if (tok_of[h] < 0 || (g & 1)) continue;
      const float f = sf.diff_gain / sqrtf(ss / static_cast<float>(DV) + sf.diff_eps);
      const int head = (head0 + (g + 8 * h) % group) / 2;
      bf16* dst = out + (static_cast<size_t>(q_begin + tok0 + tok_of[h]) * (nh / 2) + head) * DV;
#pragma unroll
      for (int dn = 0; dn < DV / 8; ++dn)
        *reinterpret_cast<uint32_t*>(dst + dn * 8 + t2) = pack_bf16(st.o[dn][2 * h] * f, st.o[dn][2 * h + 1] * f);
    }
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (tok_of[h] < 0) continue;
    const int head = head0 + (g + 8 * h) % group;
    bf16* dst = out + (static_cast<size_t>(q_begin + tok0 + tok_of[h]) * nh + head) * (kShared ? sf.out_width : DV) +
                (kShared ? sf.out_col0 : 0);
    const float l = with_sink(sf, head, st.m[h], st.l[h]);
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int dn = 0; dn < DV / 8; ++dn)
      *reinterpret_cast<uint32_t*>(dst + dn * 8 + t2) = pack_bf16(st.o[dn][2 * h] * inv, st.o[dn][2 * h + 1] * inv);
  }
}

// ------------------------------------------------------------------ launchers
constexpr size_t kSmemLimit = 226 * 1024;
constexpr size_t kQBytes = QROWS * LD * sizeof(bf16);
constexpr size_t kBarBytes = 256;
constexpr size_t kFixedBytes = 1024 + kQBytes + kBarBytes;            // alignment slack, query tile, barriers
// Six warps with two stages where that fits shared memory (head sizes up to 128), else four, else two.
constexpr int kWarps = kFixedBytes + 6 * 2 * TILE_BYTES <= kSmemLimit ? 6 : (kFixedBytes + 4 * 2 * TILE_BYTES <= kSmemLimit ? 4 : 2);
constexpr int kStages = kFixedBytes + kWarps * 3 * TILE_BYTES <= kSmemLimit ? 3 : 2;
static_assert(kFixedBytes + kWarps * kStages * TILE_BYTES <= kSmemLimit, "the key blocks must fit shared memory");
static_assert(kWarps * kStages * sizeof(uint64_t) <= kBarBytes, "barriers");
static_assert(static_cast<size_t>(kWarps + 1) * QROWS * (DV + 2) * sizeof(float) <= static_cast<size_t>(kWarps) * kStages * TILE_BYTES,
              "the merge area lies over the tiles");

B200_EXPORT int b200_attention_mma_head_dim() { return D; }
B200_EXPORT int b200_attention_mma_max_group() { return QROWS; }

B200_EXPORT int b200_kv_tensor_map(void* out_map, const void* cache, long long rows, int width, int box_rows) {
  return make_kv_tensor_map(out_map, cache, rows, width, box_rows);
}

static ScoreForm score_form(float scale, float softcap, int split_p, int chunk, const float* sinks, int v_col0,
                            int out_width, int out_col0, const float* diff) {
  ScoreForm sf;
  sf.scale_log2 = scale * 1.4426950408889634f;
  sf.tanh_in = softcap > 0.0f ? scale / softcap : 0.0f;
  sf.cap_log2 = softcap > 0.0f ? softcap * 1.4426950408889634f : 0.0f;
  sf.split_p = split_p;
  sf.chunk = chunk;
  sf.sinks = sinks;
  sf.v_col0 = v_col0;
  sf.out_width = out_width;
  sf.out_col0 = out_col0;
  sf.diff_lambda = diff != nullptr ? diff[0] : 0.0f;
  sf.diff_gain = diff != nullptr ? diff[1] : 0.0f;
  sf.diff_eps = diff != nullptr ? diff[2] : 0.0f;
  return sf;
}

// Decoded tokens over a bfloat16 cache.  `k_map`, `v_map`: descriptors from b200_kv_tensor_map with
// box_rows = min(page_size, 32); page_size must be a power of two; at most 16 query heads per KV head.
// `scratch` as for b200_decode_attention of attention.cu.
B200_EXPORT int b200_decode_attention_mma(const void* q, const void* k_map, const void* v_map, void* out,
                                          float* scratch, const int* block_table, int table_stride,
                                          const int* cu_q, const int* kv_len, const int* rows, int n_rows, int nh,
                                          int nkv, int page_size, int window, float scale, int splits,
                                          float softcap, int split_p, int chunk, const float* sinks, int v_col0,
                                          int out_width, int out_col0, const float* diff, int* err,
                                          cudaStream_t stream) {
  if (n_rows <= 0) return 0;
  if (kDiff && (diff == nullptr || sinks != nullptr || (nkv > 0 && (nh / nkv) % 2 != 0))) return B200_BAD_SIZE;
  if (nh <= 0 || nkv <= 0 || nh % nkv != 0 || nh / nkv > QROWS || page_size <= 0 || splits <= 0) return B200_BAD_SIZE;
  if ((page_size & (page_size - 1)) != 0) return B200_BAD_SIZE;
  const int box_rows = page_size < KB ? page_size : KB;
  constexpr size_t smem = kFixedBytes + static_cast<size_t>(kWarps) * kStages * TILE_BYTES;
  const bool shaped = softcap > 0.0f || split_p != 0;
  auto* kernel = shaped ? decode_mma_kernel<kWarps, kStages, true> : decode_mma_kernel<kWarps, kStages, false>;
  static bool configured[2] = {false, false};
  if (!configured[shaped]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return static_cast<int>(e);
    configured[shaped] = true;
  }
  CUtensorMap kmap, vmap;
  memcpy(&kmap, k_map, sizeof(kmap));
  memcpy(&vmap, v_map, sizeof(vmap));
  float* part_acc = scratch;
  float* part_ml = scratch + static_cast<size_t>(n_rows) * nh * splits * DV;
  dim3 grid(splits, nkv, n_rows);
  // Two, four or eight splits are the CTAs of one cluster and combine their parts through distributed shared memory;
  // other counts leave them in `scratch` for a kernel of its own.
  // (Only while the grid is one wave: clusters must be placed whole, and with several waves of one CTA per SM that
  // costs more than the second kernel, 10.1 k against 10.7 k tokens a second at batch 64.)
  static int sm_count = 0;
  if (sm_count == 0) {
    int dev = 0, n = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return static_cast<int>(e);
    sm_count = n;
  }
  const bool cluster_merge = (splits == 2 || splits == 4 || splits == 8) &&
                             static_cast<long long>(splits) * nkv * n_rows <= sm_count;
  int rc = b200_launch(kernel, grid, dim3(kWarps * 32), smem, stream, cluster_merge ? splits : 0,
                       kmap, vmap, static_cast<const bf16*>(q), static_cast<bf16*>(out), part_acc, part_ml, block_table,
                       table_stride, cu_q, kv_len, rows, nh, nkv, page_size, box_rows, window,
                       score_form(scale, softcap, split_p, chunk, sinks, v_col0, kShared ? out_width : DV, kShared ? out_col0 : 0, diff),
                       cluster_merge ? 1 : 0, err);
  if (rc != 0 || splits == 1 || cluster_merge) return rc;
  if constexpr (kDiff) {
    return b200_launch(decode_mma_merge_diff_kernel, dim3(n_rows, nh / 2), dim3(DV >= 128 ? 128 : 64), 0, stream, 0,
                       static_cast<bf16*>(out), static_cast<const float*>(part_acc), static_cast<const float*>(part_ml), cu_q,
                       rows, nh, splits, diff[0], diff[1], diff[2]);
  }
  dim3 mgrid(n_rows, nh);
  return b200_launch(decode_mma_merge_kernel, mgrid, dim3(DV >= 128 ? 128 : 64), 0, stream, 0, static_cast<bf16*>(out),
                     static_cast<const float*>(part_acc), static_cast<const float*>(part_ml), cu_q, rows, nh, splits, sinks,
                     kShared ? out_width : DV, kShared ? out_col0 : 0);
}

constexpr size_t kPfQBytes = PF_ROWS * LD * sizeof(bf16);
constexpr size_t kPfFixed = 1024 + kPfQBytes + kBarBytes;
constexpr int kPfStages = D <= 128 && DV <= 128 ? 3 : kPfFixed + 4 * TILE_BYTES <= kSmemLimit ? 4 : (kPfFixed + 3 * TILE_BYTES <= kSmemLimit ? 3 : 2);
static_assert(kPfFixed + kPfStages * TILE_BYTES <= kSmemLimit, "the key blocks must fit shared memory");

// Portions of prompts over a bfloat16 cache; arguments as b200_prefill_attention of attention.cu, with the
// descriptors of b200_kv_tensor_map in place of the cache pointers.
B200_EXPORT int b200_prefill_attention_mma(const void* q, const void* k_map, const void* v_map, void* out,
                                           const int* block_table, int table_stride, const int* cu_q,
                                           const int* kv_len, const int* prefix_len, const int* rows, int n_rows,
                                           int max_q_len, int nh, int nkv, int page_size, int window, float scale,
                                           float softcap, int split_p, int chunk, const float* sinks, int v_col0,
                                           int out_width, int out_col0, const float* diff, int* err,
                                           cudaStream_t stream) {
  if (n_rows <= 0 || max_q_len <= 0) return 0;
  if (kDiff && (diff == nullptr || sinks != nullptr || (nkv > 0 && (nh / nkv) % 2 != 0))) return B200_BAD_SIZE;
  if (nh <= 0 || nkv <= 0 || nh % nkv != 0 || nh / nkv > QROWS || page_size <= 0) return B200_BAD_SIZE;
  if ((page_size & (page_size - 1)) != 0) return B200_BAD_SIZE;
  const int box_rows = page_size < KB ? page_size : KB;
  const int tile_tokens = (16 / (nh / nkv)) * PF_WARPS;
  constexpr size_t smem = kPfFixed + static_cast<size_t>(kPfStages) * TILE_BYTES;
  const bool shaped = softcap > 0.0f || split_p != 0;
  auto* kernel = shaped ? prefill_mma_kernel<kPfStages, true> : prefill_mma_kernel<kPfStages, false>;
  static bool configured[2] = {false, false};
  if (!configured[shaped]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return static_cast<int>(e);
    configured[shaped] = true;
  }
  CUtensorMap kmap, vmap;
  memcpy(&kmap, k_map, sizeof(kmap));
  memcpy(&vmap, v_map, sizeof(vmap));
  const int n_tiles = (max_q_len + tile_tokens - 1) / tile_tokens;
  if (n_rows > 65535 || n_tiles > 65535) return B200_BAD_SIZE;      // the grid's y and z extents
  dim3 grid(nkv, n_rows, n_tiles);
  kernel<<<grid, PF_WARPS * 32, smem, stream>>>(
      kmap, vmap, static_cast<const bf16*>(q), static_cast<bf16*>(out), block_table, table_stride, cu_q, kv_len,
      prefix_len, rows, nh, nkv, page_size, box_rows, window, score_form(scale, softcap, split_p, chunk, sinks, v_col0, kShared ? out_width : DV, kShared ? out_col0 : 0, diff),
      err);
  return b200_check_launch();
}
