// Decode attention behind shared prefixes (prefix.cuh) over the bfloat16 cache, on mma.sync.  Compile with -DHEAD_DIM=<multiple of
// 16, at most 256>; pages of a power of two, at most 16 query heads a KV head.
//
// A CTA has an item: up to VT query vectors of one KV head (of a group's rows against a split of its shared keys, or one row's
// against a split of its own) and walks its keys as decode attention does (attention_mma.cu): every warp fetches blocks of 32
// keys by TMA into a ring of its own and multiplies them with 16 vectors at a time, float scores, sums and outputs in registers;
// the warps' parts are joined in shared memory.  Bound by the keys' and values' bytes; a group of more vectors than a CTA takes
// reads its shared keys once for each VT of them (from the second-level cache), which prefix_tcgen05.cu does not.
#include "attention_mma.cuh"
#include "prefix.cuh"

constexpr int NT = D <= 128 ? 2 : 1;             // sixteens of vectors (two of 256 dims do not fit a thread's registers)
constexpr int VT = 16 * NT;
#ifndef PREFIX_WARPS
#define PREFIX_WARPS (D <= 192 ? 4 : 3)
#endif
constexpr int WARPS = PREFIX_WARPS;
constexpr int MS = D + 4;                        // a vector's row where the warps' parts are joined: D outputs, maximum, sum
constexpr size_t FIXED = 1024 + VT * LD * sizeof(bf16) + 256;
#ifndef PREFIX_STAGES
#define PREFIX_STAGES (FIXED + static_cast<size_t>(WARPS) * 3 * TILE_BYTES <= 220 * 1024 ? 3 : 2)
#endif
constexpr int STAGES = PREFIX_STAGES;
constexpr size_t RING = static_cast<size_t>(WARPS) * STAGES * TILE_BYTES;
constexpr size_t JOIN = static_cast<size_t>(WARPS) * VT * MS * 4;
constexpr size_t SMEM = FIXED + (RING > JOIN ? RING : JOIN);
static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");

// The page of this lane's sub-block, inside the pool (the sink's where the table names none that is, or where the sub-block ends
// below `lowest`: those keys are another table's).
__device__ __forceinline__ int lane_page_checked(const PrefixCall& c, const PrefixItem& it, int box_rows, int first_key, int lowest, int lane) {
  if (first_key + (lane + 1) * box_rows <= lowest) return 0;
  const int page = lane_page(it.table, c.page_size, box_rows, first_key, it.end, lane);
  if (page >= 0 && page < c.pages) return page;
  atomicOr(c.err, B200_ERR_SLOT_RANGE);
  return 0;
}

// grid: the shared keys' CTAs (split, KV head, tile, group), then the rows' own (split, KV head, row).  `covered`: vectors of every
// group that another kernel serves (behind it, one CTA a KV head and group takes what is left, if anything).
__global__ void __launch_bounds__(WARPS * 32, 2)
prefix_mma_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const bf16* __restrict__ q,
                  const PrefixCall c, int box_rows, int covered) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  bf16* qs = reinterpret_cast<bf16*>(tiles + (RING > JOIN ? RING : JOIN));          // [VT][LD]
  uint64_t* bars = reinterpret_cast<uint64_t*>(qs + VT * LD);                        // [WARPS][STAGES]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < WARPS * STAGES) mbar_init(bars + threadIdx.x, 1);
  asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  __syncthreads();
  // Behind the tcgen05 kernel of the same call, which has waited for the kernels before it, this one begins beside it, and waits
  // for its end at its own: whoever waits for this kernel then waits for both.
  pdl_launch_dependents();
  if (covered == 0) pdl_wait();

  const int group = c.nh / c.nkv;
  const int cut = covered > 0 ? 1 : c.splits_shared;
  const int shared_ctas = cut * c.nkv * c.tiles * c.n_groups;
  int b = blockIdx.x;
  PrefixItem it;
  int tile = 0, tile_step = 1, last_vector;
  it.shared = b < shared_ctas;
  int lowest = 0;                                // keys below this one are not the item's
  if (it.shared) {
    const int split = b % cut;
    b /= cut;
    it.kvh = b % c.nkv;
    b /= c.nkv;
    const int2 rows = rows_of_group(c, b / c.tiles);
    const int keys = rows.y > 0 ? shared_of_group(c, b / c.tiles) : 0;
    it.i0 = rows.x;
    it.slot = split;
    it.table = c.block_table + static_cast<long long>(rows.y > 0 ? c.rows[rows.x] : 0) * c.table_stride;
    const int per = ((keys + KB - 1) / KB + cut - 1) / cut * KB;
    it.begin = min(keys, split * per);
    it.end = min(keys, it.begin + per);
    tile = covered / VT + b % c.tiles;
    tile_step = c.tiles;
    last_vector = rows.y * group;
  } else {
    b -= shared_ctas;
    const int split = b % c.splits_own;
    b /= c.splits_own;
    it.kvh = b % c.nkv;
    it.i0 = b / c.nkv;
    const int g = group_of_row(c, it.i0), row = c.rows[it.i0];
    const int keys = keys_of_row(c, row);
    lowest = min(keys, g < 0 ? 0 : shared_of_group(c, g));
    if (g < 0)                                   // (a row in front of the first group: nobody else writes its other slots)
      for (int i = threadIdx.x; i < group * c.splits_shared; i += WARPS * 32)
        c.part_ml[(static_cast<long long>(it.i0) * c.nh + it.kvh * group + i / c.splits_shared) * prefix_splits(c) + i % c.splits_shared] =
            make_float2(-INFINITY, 0.0f);
    it.table = c.block_table + static_cast<long long>(row) * c.table_stride;
    it.slot = c.splits_shared + split;
    const int from = keys > lowest ? lowest / KB * KB : keys;      // blocks begin on multiples of 32, so that no sub-block leaves its page
    const int per = ((keys - from + KB - 1) / KB + c.splits_own - 1) / c.splits_own * KB;
    it.begin = min(keys, from + split * per);
    it.end = min(keys, it.begin + per);
    last_vector = group;
  }
  const int blocks = (it.end - it.begin + KB - 1) / KB;
  const int splits = prefix_splits(c);

  unsigned char* my = tiles + static_cast<size_t>(warp) * STAGES * TILE_BYTES;
  uint64_t* my_bars = bars + warp * STAGES;
  int stage = 0;
  uint32_t parity = 0;
  ScoreForm sf = {};
  sf.scale_log2 = c.scale_log2;
  bool alive = true;                             // (a wait that ran out ends the CTA's work; what it leaves is flagged)
  for (; tile * VT < last_vector && alive; tile += tile_step) {
    it.vector0 = tile * VT;
    it.vectors = min(VT, last_vector - it.vector0);
    // the ring's first blocks; they come while the queries do
    int issue = warp;
    int page = 0, next_stage = stage;
    auto begin_next = [&]() {
      const int next = issue + WARPS;
      const int next_page = next < blocks ? lane_page_checked(c, it, box_rows, it.begin + next * KB, lowest, lane) : 0;
      if (issue < blocks) {
        fetch_block(my + next_stage * TILE_BYTES, &kmap, &vmap, page, c.page_size, c.nkv, it.kvh, box_rows, it.begin + issue * KB, it.end,
                    my_bars + next_stage, lane);
        next_stage = next_stage + 1 == STAGES ? 0 : next_stage + 1;
      }
      issue = next;
      page = next_page;
    };
    if (issue < blocks) page = lane_page_checked(c, it, box_rows, it.begin + issue * KB, lowest, lane);
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) begin_next();

    for (int x = threadIdx.x; x < VT * (D / 8); x += WARPS * 32) {
      const int r = x / (D / 8), part = x - r * (D / 8);
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (r < it.vectors) {
        const int vec = it.vector0 + r;
        const int tok = c.cu_q[c.rows[it.i0 + vec / group]];
        v = *reinterpret_cast<const uint4*>(q + (static_cast<long long>(tok) * c.nh + it.kvh * group + vec % group) * D + part * 8);
      }
      *reinterpret_cast<uint4*>(qs + r * LD + part * 8) = v;
    }
    // the last key that each of this lane's vectors sees, and the least of them among the tile's
    int last_key[2 * NT];
    int all_see = INT_MAX;
#pragma unroll
    for (int n = 0; n < 2 * NT; ++n) {
      const int r = n * 8 + (lane >> 2);
      last_key[n] = -1;
      if (r < it.vectors) {
        last_key[n] = min(it.end, keys_of_row(c, c.rows[it.i0 + (it.vector0 + r) / group])) - 1;
        all_see = min(all_see, last_key[n]);
      }
    }
    all_see = __reduce_min_sync(0xffffffffu, all_see);
    __syncthreads();
    WarpAcc st[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) st[n].init();
    for (int blk = warp; blk < blocks; blk += WARPS) {
      begin_next();
      if (!mbar_wait(my_bars + stage, parity, c.err)) {
        // Give the copies that are still in flight a bounded time to land before the tiles are used for something else.
        for (int s = 0; s < STAGES; ++s) mbar_wait(my_bars + s, s < stage ? parity ^ 1u : parity, c.err);
        alive = false;
        break;
      }
      unsigned char* t = my + stage * TILE_BYTES;
      const int first_key = it.begin + blk * KB;
      if (first_key + KB > it.end && first_key + lane >= it.end) {
        // Value rows beyond the item's keys: whatever the page holds there must not reach P.V.
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int x = 0; x < VALUE_CHUNKS; ++x) *reinterpret_cast<uint4*>(t + V_OFFSET + (x >> 3) * HALF_BYTES + lane * 128 + (x & 7) * 16) = zero;
      }
      if (first_key < lowest && first_key + lane < lowest) {
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int x = 0; x < VALUE_CHUNKS; ++x) *reinterpret_cast<uint4*>(t + V_OFFSET + (x >> 3) * HALF_BYTES + lane * 128 + (x & 7) * 16) = zero;
      }
      __syncwarp();
      const bool masked = first_key + KB - 1 > all_see || first_key < lowest;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (n * 16 >= it.vectors) break;
        const int p0 = last_key[2 * n], p1 = last_key[2 * n + 1];
        // (a row's own keys: all of its vectors end at one key, and the window reaches from there to `lowest`)
        if (masked) block_mma<true, false>(qs + n * 16 * LD, t, t + V_OFFSET, first_key, it.end, lowest > 0 ? max(p0, p1) - lowest + 1 : 0, p0, p1, sf, st[n]);
        else block_mma<false, false>(qs + n * 16 * LD, t, t + V_OFFSET, first_key, it.end, 0, p0, p1, sf, st[n]);
      }
      __syncwarp();                              // every lane is done reading before the stage is refilled
      if (++stage == STAGES) { stage = 0; parity ^= 1u; }
    }
    // The warps' parts, joined: [WARPS][VT][MS] floats over the ring.
    __syncthreads();
    float* join = reinterpret_cast<float*>(tiles);
    const int g = lane >> 2, t2 = (lane & 3) * 2;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float l = st[n].l[half];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const int r = n * 16 + g + 8 * half;
        float* dst = join + (warp * VT + r) * MS;
        if (r < it.vectors) {
#pragma unroll
          for (int dn = 0; dn < D / 8; ++dn) *reinterpret_cast<float2*>(dst + dn * 8 + t2) = make_float2(st[n].o[dn][2 * half], st[n].o[dn][2 * half + 1]);
          if ((lane & 3) == 0) { dst[D] = st[n].m[half]; dst[D + 1] = l; }
        }
      }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < it.vectors * (D / 4); x += WARPS * 32) {
      const int r = x / (D / 4), col = x - r * (D / 4);
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) m = fmaxf(m, join[(w * VT + r) * MS + D]);
      const int vec = it.vector0 + r;
      const long long place = (static_cast<long long>(it.i0 + vec / group) * c.nh + it.kvh * group + vec % group) * splits + it.slot;
      float l = 0.0f;
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (m != -INFINITY) {
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float* src = join + (w * VT + r) * MS;
          const float f = exp2f(src[D] - m);
          const float4 a = *reinterpret_cast<const float4*>(src + col * 4);
          l += src[D + 1] * f;
          o.x += a.x * f;
          o.y += a.y * f;
          o.z += a.z * f;
          o.w += a.w * f;
        }
        *reinterpret_cast<float4*>(c.part_acc + place * D + col * 4) = o;
      }
      if (col == 0) {
        c.part_ml[place] = make_float2(m, l);
        if (it.shared && covered > 0)            // (it has taken all of the keys)
          for (int s = 1; s < c.splits_shared; ++s) c.part_ml[place + s] = make_float2(-INFINITY, 0.0f);
      }
    }
    __syncthreads();                             // (a CTA may have another tile)
  }
  if (covered > 0) pdl_wait();
}

// Arguments as b200_prefix_attention, with the descriptors of b200_kv_tensor_map (attention_mma.cu; box_rows = min(page_size, 32)) in
// place of the cache.  `covered`: see the kernel; > 0: prefix_tcgen05.cu's kernel has just been launched for them.
B200_EXPORT int b200_prefix_attention_mma(const void* q, const void* k_map, const void* v_map, void* out, float* scratch, const int* block_table,
                                          int table_stride, const int* cu_q, const int* kv_len, const int* rows, int n_rows, const int* groups,
                                          int n_groups, int nh, int nkv, int page_size, int pages, float scale, int splits_shared, int splits_own,
                                          int tiles, int covered, int* err, cudaStream_t stream) {
  if (n_rows <= 0) return 0;
  if (nh <= 0 || nkv <= 0 || nh % nkv != 0 || nh / nkv > 16 || page_size <= 0 || (page_size & (page_size - 1)) != 0 || pages <= 0 || table_stride <= 0 || n_groups < 0)
    return B200_BAD_SIZE;
  if (splits_shared < 1 || splits_own < 1 || splits_shared + splits_own > 128 || tiles < 1 || covered < 0 || covered % VT != 0) return B200_BAD_SIZE;
  if (reinterpret_cast<uintptr_t>(q) % 16 != 0) return B200_BAD_ALIGN;
  const PrefixCall c = {block_table, cu_q, kv_len, rows, reinterpret_cast<const int2*>(groups), scratch,
                        reinterpret_cast<float2*>(scratch + static_cast<size_t>(n_rows) * nh * (splits_shared + splits_own) * D), err, table_stride, n_rows,
                        n_groups, nh, nkv, page_size, pages, splits_shared, splits_own, tiles, scale * 1.4426950408889634f};
  const long long ctas = static_cast<long long>(covered > 0 ? 1 : splits_shared) * nkv * tiles * n_groups + static_cast<long long>(splits_own) * nkv * n_rows;
  if (ctas > INT32_MAX) return B200_BAD_SIZE;
  static bool seen[16];
  int rc = prefix_smem_limit(prefix_mma_kernel, static_cast<int>(SMEM), seen);
  if (rc != 0) return rc;
  CUtensorMap kmap, vmap;
  memcpy(&kmap, k_map, sizeof(kmap));
  memcpy(&vmap, v_map, sizeof(vmap));
  rc = b200_launch(prefix_mma_kernel, dim3(static_cast<unsigned>(ctas)), dim3(WARPS * 32), SMEM, stream, 0, kmap, vmap, static_cast<const bf16*>(q), c,
                   page_size < KB ? page_size : KB, covered);
  if (rc != 0) return rc;
  return prefix_merge<bf16, D>(out, c, D, stream);
}
