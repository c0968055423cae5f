// The shared keys of decode attention behind prefixes (prefix.cuh) on the fifth-generation tensor cores: bfloat16, head size 128,
// groups of many rows.  A group's query vectors of one KV head (rows x query heads a KV head) are the rows of
//   S = Q K^T,  O = P V   (tcgen05.mma, M 128, blocks of 128 keys, float sums in tensor memory),
// as in the two-tile prompt kernel (attention_tcgen05.cu), whose products and softmax these are: K and V by TMA, a page's box each
// in turn, one softmax thread a row with its 128 scores in registers, the weights back into tensor memory.  Here no key is masked
// but behind a row's end, and what is stored is a split's part: float outputs, the reference maximum and the sum.
//
// A CTA has two streams, so that one's products run under the other's softmax:
//   two tiles (more than 128 vectors)   each stream has 128 vectors of its own, both walk the same keys, fetched once;
//   one tile                            both streams have the same vectors and take every other block of keys; each leaves a part
//                                       of its own, and the rings are a stage of keys deeper.
// Bound, two tiles, by the products: a pair of blocks takes 3,360 cycles, 2,050 of them products, which wait for shared memory where the
// copies write it (2,560 together); one tile by the copies' instructions, 64 of some 130 cycles a pair of blocks.  (256 vectors of 8 KV
// heads behind 32,768 keys, 13 CTAs a head: 60.7 us; with two copy warps and no more than 168 registers for the softmax, which spilled, 65.9;
// 64 vectors behind 16,384 keys 27.5 and 30.0.  Four copy warps leave 128 registers a thread: 115.5.  Scores in buffers of 64 keys, two a
// stream, ready before the softmax wants them: 65.1, for a product of 64 columns reads as many queries as one of 128.)
#include "attention_tcgen05.cuh"
#include "kv_map.cuh"
#include "prefix.cuh"

constexpr int COPY_WARPS = 3;
constexpr int THREADS = 288 + 32 * COPY_WARPS;            // warps 0-3 and 4-7 the streams' softmax, 8 products, 9-11 copies
constexpr int SOFTMAX_REGISTERS = 208, OTHER_REGISTERS = 88;      // of a thread, out of the 168 that 384 threads are launched with
static_assert(256 * SOFTMAX_REGISTERS + (THREADS - 256) * OTHER_REGISTERS <= THREADS * 168, "the split is of what the launch has");
constexpr int V_STAGES = 2;
constexpr int V_OFF = 0, Q_OFF = V_STAGES * TILE, K_OFF_TWO = Q_OFF + 2 * TILE, K_OFF_ONE = Q_OFF + TILE;
constexpr int BAR_OFF = 6 * TILE;                         // V 2, Q 2 and K 2, or V 2, Q 1 and K 3
constexpr int OUT_PITCH = D * 4 + 16;                      // of a row of outputs in shared memory
static_assert(256 * OUT_PITCH <= BAR_OFF, "the outputs' rows fit where the tiles were");
constexpr int N_BARS = 2 * 3 + 2 * V_STAGES + 4 * 2 + 1;
constexpr int TBL_OFF = BAR_OFF + (N_BARS + 1) * 8;
constexpr int SMEM = 1024 + TBL_OFF + TBL_ENTRIES * 4;
static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");

// grid (splits' CTAs, KV heads, groups * tiles of 128 or 256 vectors).
template <bool TWO>
__global__ void __launch_bounds__(THREADS, 1)
prefix_tcgen05_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const bf16* __restrict__ q,
                      const PrefixCall c, int box_rows) {
  constexpr int KS = TWO ? 2 : 3, VS = V_STAGES, K_OFF = TWO ? K_OFF_TWO : K_OFF_ONE;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(sm + BAR_OFF);
  uint64_t* k_empty = k_full + 3;
  uint64_t* v_full = k_empty + 3;
  uint64_t* v_empty = v_full + VS;
  uint64_t* s_full = v_empty + VS;                                   // [2]: one a stream, and so on
  uint64_t* p_full = s_full + 2;
  uint64_t* p_half = p_full + 2;
  uint64_t* pv_done = p_half + 2;
  uint64_t* q_full = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 1);

  const int warp = same_in_warp(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x < 32) prefetch_indices(c);
  if (threadIdx.x == 0) {
    for (int s = 0; s < 3; ++s) { mbar_init(k_full + s, 1); mbar_init(k_empty + s, 1); }
    for (int s = 0; s < VS; ++s) { mbar_init(v_full + s, 1); mbar_init(v_empty + s, 1); }
    for (int t = 0; t < 2; ++t) { mbar_init(s_full + t, 1); mbar_init(p_full + t, 4); mbar_init(p_half + t, 4); mbar_init(pv_done + t, 1); }
    mbar_init(q_full, TWO ? 8 : 4);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = same_in_warp(*tmem_slot);        // columns: S of stream 0 0..127, of stream 1 128..255, O 256..383 and 384..511
  // The kernel behind this one in the call (prefix_mma.cu's, the rows' own keys) does not read what this one writes and may run beside
  // it, but what was launched before this one must have ended: so first the wait, then the word.
  pdl_wait();
  pdl_launch_dependents();

  const int kvh = blockIdx.y, g = blockIdx.z / c.tiles, tile = blockIdx.z % c.tiles;
  const int group = c.nh / c.nkv;
  const int2 rows = rows_of_group(c, g);
  const int vector0 = tile * (TWO ? 2 * BQ : BQ);
  const int vectors = max(0, min(TWO ? 2 * BQ : BQ, rows.y * group - vector0));
  // CTA x takes blocks [first, first + count) of the shared keys; its streams' slots are x (two tiles) or 2x and 2x + 1.
  const int keys = vectors > 0 ? shared_of_group(c, g) : 0;
  const int blocks = (keys + BKV - 1) / BKV;
  const int per = (blocks + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  const int first = min(blocks, static_cast<int>(blockIdx.x) * per);
  const int count = same_in_warp(min(blocks, first + per) - first);
  const int k_begin = first * BKV, k_end = min(keys, k_begin + count * BKV);
  // the streams' blocks: block j of stream t is the CTA's block j, or 2j + t
  const int nblk[2] = {TWO ? count : (count + 1) / 2, TWO ? (vectors > BQ ? count : 0) : count / 2};
  const int* table = c.block_table + static_cast<long long>(rows.y > 0 ? c.rows[rows.x] : 0) * c.table_stride;

  if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(OTHER_REGISTERS));
  else asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(SOFTMAX_REGISTERS));
  if (warp > 8) {
    // ---- copies, as in the prompt kernels: the page numbers first, then the blocks' boxes, COPY_WARPS warps in turn
    const int cw = warp - 9;
    bool ok = true;
    int* tbl = reinterpret_cast<int*>(sm + TBL_OFF);
    const int first_page = k_begin / c.page_size;
    const int n_pages = min(TBL_ENTRIES, (k_end + c.page_size - 1) / c.page_size - first_page);
    auto checked = [&](int page) {                               // (the sink's page where the table names none of the pool's)
      if (page >= 0 && page < c.pages) return page;
      atomicOr(c.err, B200_ERR_SLOT_RANGE);
      return 0;
    };
    for (int t = cw * 32 + lane; t < n_pages; t += 32 * COPY_WARPS) tbl[t] = checked(table[first_page + t]);
    asm volatile("bar.sync 1, %0;\n" ::"n"(32 * COPY_WARPS) : "memory");      // (the copy warps only)
    auto fetch = [&](const CUtensorMap* map, unsigned char* dst, uint64_t* bar, int first_key) {
      const int n_sub = (min(BKV, k_end - first_key) + box_rows - 1) / box_rows;
      proxy_fence();
      if (cw == 0 && lane == 0) mbar_expect_tx(bar, static_cast<uint32_t>(n_sub) * 2u * box_rows * 128u);
      __syncwarp();
      for (int j = cw + COPY_WARPS * lane; j < n_sub; j += 32 * COPY_WARPS) {
        const int key0 = first_key + j * box_rows;
        const int pi = key0 / c.page_size - first_page;
        const int page = pi < TBL_ENTRIES ? tbl[pi] : checked(table[first_page + pi]);
        const int y = (page * c.nkv + kvh) * c.page_size + key0 % c.page_size;
        tma_load_2d(dst + j * box_rows * 128, map, 0, y, bar);
        tma_load_2d(dst + HALF + j * box_rows * 128, map, 64, y, bar);
      }
    };
    int ik = 0;
    for (int i = 0; i < count && ok; ++i) {
      for (; ik < count && ik <= i + KS - 1 && ok; ++ik) {
        const int s = ik % KS, use = ik / KS;
        if (use > 0) ok = mbar_wait_warp(k_empty + s, (use - 1) & 1, c.err);
        if (ok) fetch(&kmap, sm + K_OFF + s * TILE, k_full + s, k_begin + ik * BKV);
      }
      if (!ok) break;
      const int s = i % VS, use = i / VS;
      if (use > 0) ok = mbar_wait_warp(v_empty + s, (use - 1) & 1, c.err);
      if (ok) fetch(&vmap, sm + V_OFF + s * TILE, v_full + s, k_begin + i * BKV);
    }
  } else if (warp == 8) {
    // ---- products: P V of a stream's block, then S of its next one, the streams in turn
    if (count > 0) {
      bool ok = mbar_wait_warp(q_full, 0, c.err);
      const uint64_t dq = desc_k_major(smem_u32(sm + Q_OFF)), dk = desc_k_major(smem_u32(sm + K_OFF)), dv = desc_mn_major(smem_u32(sm + V_OFF));
      auto block_of = [&](int t, int j) { return TWO ? j : 2 * j + t; };
      auto last_user = [&](int t) { return !TWO || t == 1 || nblk[1] == 0; };      // (of a block: two tiles use it one after the other)
      auto issue_s = [&](int t, int j) {
        const int i = block_of(t, j), s = i % KS;
        if (!mbar_wait_warp(k_full + s, (i / KS) & 1, c.err)) return false;
        tc_fence_after();
        const uint64_t q0 = dq + static_cast<uint32_t>(TWO ? t * (TILE >> 4) : 0), k0 = dk + static_cast<uint32_t>(s * (TILE >> 4));
        if (elect_one()) {
#pragma unroll
          for (int x = 0; x < D / 16; ++x) {
            const uint32_t off = ((x >> 2) * HALF + (x & 3) * 32) >> 4;
            umma(tmem_base + t * 128, q0 + off, k0 + off, kDescQK, x > 0 ? 1u : 0u);
          }
          umma_commit(s_full + t);
          if (last_user(t)) umma_commit(k_empty + s);
        }
        __syncwarp();
        return true;
      };
      if (ok && nblk[0] > 0) ok = issue_s(0, 0);
      if (ok && nblk[1] > 0) ok = issue_s(1, 0);
      for (int j = 0; j < nblk[0] && ok; ++j) {                      // (stream 0 has as many blocks as stream 1, or one more)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!ok || j >= nblk[t]) continue;
          const int i = block_of(t, j), s = i % VS;
          ok = mbar_wait_warp(p_half + t, j & 1, c.err);             // P lies where S lay
          if (ok) ok = mbar_wait_warp(v_full + s, (i / VS) & 1, c.err);
          if (!ok) continue;
          tc_fence_after();
          const uint64_t v0 = dv + static_cast<uint32_t>(s * (TILE >> 4));
          const uint32_t tmem_o = tmem_base + 256 + t * 128, tmem_p = tmem_base + t * 128, more = j > 0 ? 1u : 0u;
          if (elect_one()) {
#pragma unroll
            for (int x = 0; x < BKV / 32; ++x) umma_a_tmem(tmem_o, tmem_p + x * 8, v0 + x * 128, kDescPV, x > 0 ? 1u : more);
          }
          __syncwarp();
          ok = mbar_wait_warp(p_full + t, j & 1, c.err);
          if (!ok) continue;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int x = BKV / 32; x < BKV / 16; ++x) umma_a_tmem(tmem_o, tmem_p + x * 8, v0 + x * 128, kDescPV, 1u);
            umma_commit(pv_done + t);
            if (last_user(t)) umma_commit(v_empty + s);
          }
          __syncwarp();
          if (j + 1 < nblk[t]) ok = issue_s(t, j + 1);
        }
      }
    }
  } else {
    // ---- softmax: thread (stream t, row r) owns one query vector (tensor-memory lane r of the stream's columns)
    const int t = warp >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const int vec = vector0 + (TWO ? t * BQ : 0) + r;
    const bool used = vec - vector0 < vectors;
    const int row = rows.x + vec / group, head = kvh * group + vec % group;
    int hi_key = -1, batch_row = 0;
    if (used) {
      batch_row = c.rows[row];
      hi_key = min(k_end, keys_of_row(c, batch_row)) - 1;
    }
    if (count > 0 && (TWO || t == 0)) {
      // The warp's 32 vectors, half a warp a vector, all on their way at once (zeros where there is none).  (Each lane its own vector,
      // 32 lines an instruction: 5,700 cycles.)
      const long long mine_at = used ? (static_cast<long long>(c.cu_q[batch_row]) * c.nh + head) * D : -1;
      uint4 v[16];
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const long long at = __shfl_sync(0xffffffffu, mine_at, 2 * x + (lane >> 4));
        v[x] = make_uint4(0u, 0u, 0u, 0u);
        if (at >= 0) v[x] = *reinterpret_cast<const uint4*>(q + at + (lane & 15) * 8);
      }
#pragma unroll
      for (int x = 0; x < 16; ++x) *reinterpret_cast<uint4*>(sm + Q_OFF + t * TILE + swz(quarter * 32 + 2 * x + (lane >> 4), lane & 15)) = v[x];
      proxy_fence();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    // the least of the last keys that this warp's vectors see
    const int all_see = __reduce_min_sync(0xffffffffu, used ? hi_key : INT_MAX);
    RowState st;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t s_base = lane_base + t * 128, o_base = lane_base + 256 + t * 128;
    const int mine = t ? nblk[1] : nblk[0];
    bool ok = true;
    for (int j = 0; j < mine; ++j) {
      const int i = TWO ? j : 2 * j + t;
      const int first_key = k_begin + i * BKV;
      if (!mbar_wait_warp(s_full + t, j & 1, c.err)) { ok = false; break; }
      // Value rows beyond the keys must not reach P V, whatever the page or the stage held (two tiles write the same zeros,
      // each before its own product).
      if (first_key + BKV > k_end) {
        const int s = i % VS;
        ok = mbar_wait_warp(v_full + s, (i / VS) & 1, c.err);
        if (!ok) break;
        if (first_key + r >= k_end) zero_value_row<16>(sm + V_OFF + s * TILE, r, 0);
        proxy_fence();
      }
      softmax_row(s_base, o_base, first_key, 0, hi_key, first_key + BKV - 1 > all_see, c.scale_log2, j, st, [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_half + t);
      });
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + t);
    }
    // (S of the last block was issued behind P V of the one before it: only this phase can be the one that runs)
    if (ok && mine > 0) ok = mbar_wait_warp(pv_done + t, (mine - 1) & 1, c.err);
    const int slot = TWO ? static_cast<int>(blockIdx.x) : 2 * static_cast<int>(blockIdx.x) + t;
    const long long place = (static_cast<long long>(row) * c.nh + head) * prefix_splits(c) + slot;
    const bool seen = ok && mine > 0 && (st.m_ref > -INFINITY || st.l_run != st.l_run);
    if (used) c.part_ml[place] = seen ? part_of(st.m_ref, st.l_run) : make_float2(-INFINITY, 0.0f);
    // The outputs leave through shared memory, where both streams' products have been done: a thread puts its row there (rows 528
    // bytes apart, so that eight threads' pieces lie in eight different groups of banks) and the copy engine takes it.  (Straight
    // from the registers, 32 lines an instruction: 6,000 to 9,000 cycles.)
    asm volatile("bar.sync 2, 256;\n" ::: "memory");             // (the softmax warps, whatever became of their waits)
    if (ok && mine > 0) {
      tc_fence_after();
      unsigned char* line = sm + threadIdx.x * OUT_PITCH;
#pragma unroll 1
      for (int x = 0; x < 4; ++x) {
        float o[32];
        tmem_ld32(o_base + x * 32, o);
#pragma unroll
        for (int e = 0; e < 8; ++e) *reinterpret_cast<float4*>(line + x * 128 + e * 16) = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
      }
      proxy_fence();
      if (used && seen) {
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n" ::"l"(c.part_acc + place * D), "r"(smem_u32(line)), "n"(D * 4) : "memory");
        asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
        asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
      }
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

// The first tiles % 2^16 tiles (of one or `two` times 128) of every one of the first tiles / 2^16 groups' vectors (0: of all groups')
// against its shared keys, whose parts go to slots 0 .. splits_shared - 1 of [n_rows * nh][splits_shared], at the start of `scratch`
// (splits_shared is the number of CTAs, or with one tile a CTA twice that).  The kernels of b200_prefix_attention_mma follow.  Other arguments as
// there.  (CTAs of a group that shares nothing stand in the way of the stream kernel's, an SM each: one group of 64 rows behind 32,768 keys and an
// empty one 79.4 us, without them 67.7; 24 rows of 64 heads behind 8,000 45.2 and 34.4.)
B200_EXPORT int b200_prefix_tcgen05(const void* q, const void* k_cache, const void* v_cache, float* scratch, const int* block_table, int table_stride,
                                    const int* cu_q, const int* kv_len, const int* rows, int n_rows, const int* groups, int n_groups, int nh, int nkv,
                                    int page_size, int pages, float scale, int splits_shared, int tiles, int two, int* err,
                                    cudaStream_t stream) {
  if (n_rows <= 0 || n_groups <= 0) return 0;
  if (nh <= 0 || nkv <= 0 || nkv > 65535 || nh % nkv != 0 || page_size <= 0 || (page_size & (page_size - 1)) != 0 || pages <= 0 || table_stride <= 0) return B200_BAD_SIZE;
  const int served = tiles >> 16 == 0 ? n_groups : tiles >> 16;
  tiles &= 0xffff;
  if (splits_shared < 1 || tiles < 1 || served < 1 || served > n_groups || (two == 0 && splits_shared % 2 != 0) ||
      static_cast<long long>(served) * tiles > 65535)
    return B200_BAD_SIZE;
  if (!prefix_can_be_served({q, k_cache, v_cache, scratch, block_table, cu_q, kv_len, rows, err}, groups, n_groups, table_stride, page_size))
    return B200_BAD_SIZE;
  if (static_cast<long long>(pages) * nkv * page_size > INT32_MAX) return B200_BAD_SIZE;      // (a copy's row is counted in 32 bits)
  if (!(scale > 0.0f)) return B200_BAD_SIZE;                         // maxima and masks are taken of the unscaled scores
  if (reinterpret_cast<uintptr_t>(q) % 16 != 0) return B200_BAD_ALIGN;
  const PrefixCall c = {block_table, cu_q, kv_len, rows, reinterpret_cast<const int2*>(groups), scratch,
                        reinterpret_cast<float2*>(scratch + static_cast<size_t>(n_rows) * nh * splits_shared * D), err, table_stride, n_rows,
                        n_groups, nh, nkv, page_size, pages, splits_shared, 0, tiles, scale * 1.4426950408889634f};
  static bool seen[2][16];
  auto* kernel = two != 0 ? prefix_tcgen05_kernel<true> : prefix_tcgen05_kernel<false>;
  CUtensorMap kmap, vmap;
  const int box_rows = page_size < 32 ? page_size : 32;
  const long long lines = static_cast<long long>(pages) * nkv * page_size;
  int rc = make_kv_tensor_map(&kmap, k_cache, lines, D, box_rows);
  if (rc == 0) rc = make_kv_tensor_map(&vmap, v_cache, lines, D, box_rows);
  if (rc == 0) rc = prefix_smem_limit(kernel, SMEM, seen[two != 0]);
  if (rc != 0) return rc;
  return b200_launch(kernel, dim3(two != 0 ? splits_shared : splits_shared / 2, nkv, served * tiles), dim3(THREADS), SMEM, stream, 0, kmap, vmap,
                     static_cast<const bf16*>(q), c, box_rows);
}
