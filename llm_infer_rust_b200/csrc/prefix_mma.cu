// Decode attention behind shared prefixes (prefix.cuh) over the bfloat16 cache, on mma.sync.  Compile with -DHEAD_DIM=<multiple of
// 16, at most 256>; pages of a power of two, at most 16 query heads a KV head.
//
// Work comes in items: up to 16 query vectors of one KV head (a tile of a group's against its shared keys, or one row's against its
// own), an item in blocks of 32 keys.  All items' blocks stand in one sequence, and every warp of a persistent grid takes an equal
// stretch of it, whatever the rows' lengths.  A warp works alone: it fetches blocks by TMA into a ring of its own, across the
// borders of items, multiplies them (as attention_mma.cu does) with an item's queries, which stay in registers up to 128 dims and come
// while the item before is worked on, and leaves for each item that it touches one part: float outputs, maximum, sum.  Stretch w
// and item x meet in part w + x, which rises along the sequence, so no two meet in one place and none needs to be asked for.
// A kernel behind this one joins a vector's parts.
//
// Bound by the keys' and values' bytes.  (A CTA an item with a split, warps joined in shared memory: 64 rows of 1 to 1,024 own keys, 8 KV
// heads, took 52 us, 2.6 TB/s, most of it the CTAs' beginnings and ends.)  A group of more than 16 vectors reads its shared keys
// once for each 16 (from the second-level cache), which prefix_tcgen05.cu does not.
#include "attention_mma.cuh"
#include "kv_map.cuh"
#include "prefix.cuh"

constexpr bool kQueriesInRegisters = D <= 128;
constexpr int VT = 16;                           // query vectors of an item
constexpr int STAGES = 2;
constexpr int WARPS = D <= 64 ? 8 : D <= 128 ? 6 : D <= 192 ? 4 : 3;
constexpr int THREADS = WARPS * 32;
constexpr int MOST_ENTRIES = 400;                // rows and groups of a call, whose places in the sequence stand in shared memory
constexpr size_t RING = static_cast<size_t>(WARPS) * STAGES * TILE_BYTES;
constexpr size_t QUERIES = static_cast<size_t>(WARPS) * VT * LD * sizeof(bf16);

// A group's or a row's place in the sequence of blocks (of one KV head).
struct Entries {
  int start[MOST_ENTRIES + 1];                   // its first block
  int keys[MOST_ENTRIES];                        // a group's shared keys, a row's keys
  int low[MOST_ENTRIES];                         // a group's first row; a row's first own key
  int where[MOST_ENTRIES];                       // the tiles of the groups before; a row's place in the block table
  int token[MOST_ENTRIES];                       // a row's token
  int sums[WARPS + 1];
};
constexpr size_t SMEM = 1024 + RING + QUERIES + sizeof(Entries) + WARPS * STAGES * 8;
static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");

// What the joining kernel has to know of the sequence (in device memory, written by the first CTA).
struct Sequence {
  int blocks;                                    // of one KV head
  int items;                                     // of one KV head
  int workers;
  int group_tiles;                               // of all groups
  int start[MOST_ENTRIES + 1];
  int tiles_before[MOST_ENTRIES];
};

struct StreamCall {
  PrefixCall c;                                  // part_acc, part_ml: of the tcgen05 kernel, [n_rows * nh][splits_shared]
  float* acc;                                    // [parts][16][D]
  float2* ml;                                    // [parts][16]
  Sequence* sequence;
  int covered;                                   // vectors of each group that the tcgen05 kernel serves
};

__device__ __forceinline__ int tiles_of(const StreamCall& k, int rows, int group) { return (max(0, rows * group - k.covered) + VT - 1) / VT; }

// The stretch that block s of the whole sequence is in: stretch w begins at block floor(w total / workers).
__device__ __forceinline__ int worker_of(long long s, long long total, int workers) { return static_cast<int>(((s + 1) * workers - 1) / total); }

// Where a worker stands: `left` blocks of an item from key first_key on.
struct Place {
  long long s;
  int kvh, first_key, end, lowest, left, item, i0, vector0, vectors, table_row;
  bool shared;
};

// The page of this lane's sub-block, inside the pool (the sink's where the table names none that is, or where the sub-block ends
// below `lowest`: those keys are another table's).
__device__ __forceinline__ int lane_page_checked(const PrefixCall& c, const Place& p, int box_rows, int lane) {
  const int key0 = p.first_key + lane * box_rows;
  if (lane * box_rows >= KB || key0 >= p.end || key0 + box_rows <= p.lowest) return 0;
  const int page = c.block_table[static_cast<long long>(p.table_row) * c.table_stride + key0 / c.page_size];
  if (page >= 0 && page < c.pages) return page;
  atomicOr(c.err, B200_ERR_SLOT_RANGE);
  return 0;
}

// One block of 32 keys against the 16 vectors whose queries are `qa` (or stand at `qs`): as block_mma of attention_mma.cuh, with the
// last key that a vector sees (last0, last1: of rows lane / 4 and lane / 4 + 8; -1: none) and the item's first.
template <bool MASKED>
__device__ __forceinline__ void item_block(const uint32_t (&qa)[kQueriesInRegisters ? D / 16 : 1][4], const bf16* qs, const unsigned char* ks,
                                           const unsigned char* vs, int first_key, int lowest, int last0, int last1, float scale_log2, WarpAcc& st) {
  const int lane = threadIdx.x & 31;
  const int mi = lane >> 3, r8 = lane & 7;
  float s[4][4];
#pragma unroll
  for (int n = 0; n < 4; ++n) { s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f; }
#pragma unroll
  for (int k16 = 0; k16 < D / 16; ++k16) {
    uint32_t a[4];
    if constexpr (kQueriesInRegisters) {
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = qa[k16][e];
    } else {
      ldmatrix_x4(a, qs + (lane & 15) * LD + k16 * 16 + (lane >> 4) * 8);
    }
#pragma unroll
    for (int n = 0; n < 4; n += 2) {
      uint32_t b[4];
      ldmatrix_x4(b, ks + swz(n * 8 + (mi >> 1) * 8 + r8, k16 * 2 + (mi & 1)));
      mma_bf16(s[n], a, b[0], b[1]);
      mma_bf16(s[n + 1], a, b[2], b[3]);
    }
  }
  const int t2 = (lane & 3) * 2;
  float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (MASKED) {
        const int key = first_key + n * 8 + t2 + e;
        s[n][e] = key >= lowest && key <= last0 ? s[n][e] * scale_log2 : -INFINITY;
        s[n][2 + e] = key >= lowest && key <= last1 ? s[n][2 + e] * scale_log2 : -INFINITY;
      } else {
        s[n][e] *= scale_log2;
        s[n][2 + e] *= scale_log2;
      }
      mx0 = fmaxf(mx0, s[n][e]);
      mx1 = fmaxf(mx1, s[n][2 + e]);
    }
  }
  mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1)); mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
  mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1)); mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
  const float m0 = fmaxf(st.m[0], mx0), m1 = fmaxf(st.m[1], mx1);
  const float base0 = m0 == -INFINITY ? 0.0f : m0, base1 = m1 == -INFINITY ? 0.0f : m1;
  const float c0 = fast_exp2(st.m[0] - base0), c1 = fast_exp2(st.m[1] - base1);       // (0 on the first visible block)
  float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      s[n][e] = fast_exp2(s[n][e] - base0);
      s[n][2 + e] = fast_exp2(s[n][2 + e] - base1);
      sum0 += s[n][e];
      sum1 += s[n][2 + e];
    }
  }
  const bool moved = m0 != st.m[0] || m1 != st.m[1];
  st.m[0] = m0; st.m[1] = m1;
  st.l[0] = st.l[0] * c0 + sum0;
  st.l[1] = st.l[1] * c1 + sum1;
  if (__any_sync(0xffffffffu, moved)) {            // (no row's maximum moved: nothing to rescale)
#pragma unroll
    for (int i = 0; i < D / 8; ++i) { st.o[i][0] *= c0; st.o[i][1] *= c0; st.o[i][2] *= c1; st.o[i][3] *= c1; }
  }
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    // a weight is rounded to bfloat16 once, as the A operand of P V (the values are bfloat16 themselves)
    const uint32_t a[4] = {pack_bf16(s[2 * kk][0], s[2 * kk][1]), pack_bf16(s[2 * kk][2], s[2 * kk][3]),
                           pack_bf16(s[2 * kk + 1][0], s[2 * kk + 1][1]), pack_bf16(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
    for (int dn = 0; dn < D / 8; dn += 2) {
      uint32_t b[4];
      ldmatrix_x4_trans(b, vs + swz(kk * 16 + (mi & 1) * 8 + r8, dn + (mi >> 1)));
      mma_bf16(st.o[dn], a, b[0], b[1]);
      mma_bf16(st.o[dn + 1], a, b[2], b[3]);
    }
  }
}

__global__ void __launch_bounds__(THREADS, 1)
prefix_stream_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const bf16* __restrict__ q,
                     const StreamCall k, int box_rows) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  bf16* queries = reinterpret_cast<bf16*>(tiles + RING);
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<unsigned char*>(queries) + QUERIES);      // [WARPS][STAGES]
  Entries& at = *reinterpret_cast<Entries*>(bars + WARPS * STAGES);
  const PrefixCall& c = k.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < WARPS * STAGES) mbar_init(bars + threadIdx.x, 1);
  asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  // Behind the tcgen05 kernel of the same call, which has waited for the kernels before it, this one begins beside it, and waits
  // for its end at its own: whoever waits for this kernel then waits for both.
  pdl_launch_dependents();
  if (k.covered == 0) pdl_wait();

  // ---- the sequence: groups, then rows
  const int group = c.nh / c.nkv;
  const int n_entries = c.n_groups + c.n_rows;
  for (int g = threadIdx.x; g < c.n_groups; g += THREADS) {
    const int2 rows = rows_of_group(c, g);
    at.keys[g] = rows.y > 0 ? shared_of_group(c, g) : 0;
    at.low[g] = rows.x;
    at.where[g] = tiles_of(k, rows.y, group);
  }
  for (int i = threadIdx.x; i < c.n_rows; i += THREADS) {
    const int e = c.n_groups + i, row = c.rows[i];
    at.where[e] = row;
    at.keys[e] = keys_of_row(c, row);
    at.token[e] = c.cu_q[row];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < c.n_rows; i += THREADS) {
    int lo = 0, hi = c.n_groups;                   // the groups that begin at or before row i
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (at.low[mid] <= i) lo = mid + 1; else hi = mid;
    }
    // (groups that begin at one row: the last of them has it)
    at.low[c.n_groups + i] = lo == 0 ? 0 : min(at.keys[c.n_groups + i], at.keys[lo - 1]);
  }
  __syncthreads();
  auto blocks_of = [&](int e) {
    if (e < c.n_groups) return at.where[e] * ((at.keys[e] + KB - 1) / KB);
    return at.keys[e] > at.low[e] ? (at.keys[e] + KB - 1) / KB - at.low[e] / KB : 0;
  };
  // exclusive sums: a thread's own stretch of the entries, then the warps', then the CTA's
  const int each = (n_entries + THREADS - 1) / THREADS, e0 = min(n_entries, static_cast<int>(threadIdx.x) * each), e1 = min(n_entries, e0 + each);
  int mine = 0;
  for (int e = e0; e < e1; ++e) mine += blocks_of(e);
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int before = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += before;
  }
  if (lane == 31) at.sums[warp] = upto;
  __syncthreads();
  int sum = upto - mine;
  for (int w = 0; w < warp; ++w) sum += at.sums[w];
  for (int e = e0; e < e1; ++e) {
    at.start[e] = sum;
    sum += blocks_of(e);
  }
  if (e0 < n_entries && e1 == n_entries) at.start[n_entries] = sum;
  __syncthreads();
  if (warp == 0) {                                 // the tiles of the groups before each one
    int before = 0;
    for (int g0 = 0; g0 < c.n_groups; g0 += 32) {
      const int here = g0 + lane < c.n_groups ? at.where[g0 + lane] : 0;
      int tiles_upto = here;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int less = __shfl_up_sync(0xffffffffu, tiles_upto, o);
        if (lane >= o) tiles_upto += less;
      }
      if (g0 + lane < c.n_groups) at.where[g0 + lane] = before + tiles_upto - here;
      before += __shfl_sync(0xffffffffu, tiles_upto, 31);
    }
    if (lane == 0) at.sums[WARPS] = before;
  }
  __syncthreads();
  const int blocks = at.start[n_entries], group_tiles = at.sums[WARPS], items = group_tiles + c.n_rows;
  const long long total = static_cast<long long>(blocks) * c.nkv;
  const int workers = static_cast<int>(min(static_cast<long long>(gridDim.x) * WARPS, max(total, 1ll)));
  if (blockIdx.x == 0) {
    for (int e = threadIdx.x; e <= n_entries; e += THREADS) k.sequence->start[e] = at.start[e];
    for (int g = threadIdx.x; g < c.n_groups; g += THREADS) k.sequence->tiles_before[g] = at.where[g];
    if (threadIdx.x == 0) {
      k.sequence->blocks = blocks;
      k.sequence->items = items;
      k.sequence->workers = workers;
      k.sequence->group_tiles = group_tiles;
    }
  }

  const int worker = warp * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x);      // (few stretches: on as many SMs as can be)
  const long long s_end = worker < workers ? (worker + 1) * total / workers : 0;
  auto locate = [&](long long s) {
    Place p;
    p.s = s;
    p.kvh = static_cast<int>(s / blocks);
    const int pos = static_cast<int>(s - static_cast<long long>(p.kvh) * blocks);
    int lo = 0, hi = n_entries;                    // the entries that begin at or before pos: the last of them holds it
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (at.start[mid] <= pos) lo = mid + 1; else hi = mid;
    }
    const int e = lo - 1;
    int block = pos - at.start[e], of;
    p.shared = e < c.n_groups;
    p.end = at.keys[e];
    if (p.shared) {
      of = (p.end + KB - 1) / KB;
      const int tile = block / of;
      block -= tile * of;
      p.item = p.kvh * items + at.where[e] + tile;
      p.lowest = 0;
      p.i0 = at.low[e];
      const int next = e + 1 < c.n_groups ? max(at.low[e + 1], p.i0) : c.n_rows;
      p.vector0 = k.covered + tile * VT;
      p.vectors = min(VT, (next - p.i0) * group - p.vector0);
      p.table_row = at.where[c.n_groups + p.i0];
      p.first_key = block * KB;
    } else {
      p.lowest = at.low[e];
      of = (p.end + KB - 1) / KB - p.lowest / KB;
      p.item = p.kvh * items + group_tiles + e - c.n_groups;
      p.i0 = e - c.n_groups;
      p.vector0 = 0;
      p.vectors = group;
      p.table_row = at.where[e];
      p.first_key = (p.lowest / KB + block) * KB;
    }
    p.left = static_cast<int>(min(static_cast<long long>(of - block), s_end - s));
    return p;
  };

  long long s = worker < workers ? worker * total / workers : 0;
  if (s < s_end) {
    unsigned char* ring = tiles + static_cast<size_t>(warp) * STAGES * TILE_BYTES;
    uint64_t* full = bars + warp * STAGES;
    bf16* qs = queries + warp * VT * LD;
    // the queries of an item into shared memory
    auto fetch_queries = [&](const Place& p) {
      for (int x = lane; x < VT * (D / 8); x += 32) {
        const int r = x / (D / 8), part = x - r * (D / 8);
        const int vec = p.vector0 + min(r, p.vectors - 1);
        const int token = at.token[c.n_groups + p.i0 + vec / group];
        cp_async16(qs + r * LD + part * 8, q + (static_cast<long long>(token) * c.nh + p.kvh * group + vec % group) * D + part * 8, r < p.vectors);
      }
      cp_async_commit();
    };
    Place now = locate(s), ahead = now;
    int page = lane_page_checked(c, ahead, box_rows, lane);
    int fetch_stage = 0;
    // The next block of the stretch on its way, whatever item it is of; the page numbers of the one behind it are asked for.
    auto fetch_next = [&]() {
      if (ahead.s >= s_end) return;
      fetch_block(ring + fetch_stage * TILE_BYTES, &kmap, &vmap, page, c.page_size, c.nkv, ahead.kvh, box_rows, ahead.first_key, ahead.end, full + fetch_stage, lane);
      fetch_stage = fetch_stage + 1 == STAGES ? 0 : fetch_stage + 1;
      ++ahead.s;
      ahead.first_key += KB;
      if (--ahead.left == 0 && ahead.s < s_end) ahead = locate(ahead.s);
      if (ahead.s < s_end) page = lane_page_checked(c, ahead, box_rows, lane);
    };
    fetch_queries(now);
#pragma unroll
    for (int x = 0; x < STAGES - 1; ++x) fetch_next();
    int stage = 0;
    uint32_t parity = 0;
    bool alive = true;                             // (a wait that ran out ends the warp's work; the error word says so)
    while (alive) {
      uint32_t qa[kQueriesInRegisters ? D / 16 : 1][4];
      cp_async_wait<0>();
      __syncwarp();
      const long long behind = now.s + now.left;
      Place next = now;
      if constexpr (kQueriesInRegisters) {
#pragma unroll
        for (int x = 0; x < D / 16; ++x) ldmatrix_x4(qa[x], qs + (lane & 15) * LD + x * 16 + (lane >> 4) * 8);
        __syncwarp();
        if (behind < s_end) {
          next = locate(behind);
          fetch_queries(next);
        }
      }
      // the last key that this lane's two vectors see, and the least of all vectors'
      int last[2], all_see = INT_MAX;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = x * 8 + (lane >> 2);
        last[x] = -1;
        if (r < now.vectors) {
          last[x] = min(now.end, at.keys[c.n_groups + now.i0 + (now.vector0 + r) / group]) - 1;
          all_see = min(all_see, last[x]);
        }
      }
      all_see = __reduce_min_sync(0xffffffffu, all_see);
      WarpAcc st;
      st.init();
      for (int x = 0; x < now.left; ++x) {
        fetch_next();
        if (!mbar_wait(full + stage, parity, c.err)) {
          // Give the copies that are still in flight a bounded time to land before the warp leaves.
          for (int t = 0; t < STAGES; ++t) mbar_wait(full + t, t < stage ? parity ^ 1u : parity, c.err);
          alive = false;
          break;
        }
        unsigned char* t = ring + stage * TILE_BYTES;
        const int first_key = now.first_key + x * KB;
        if (first_key + KB > now.end || first_key < now.lowest) {
          // Value rows that are not the item's: whatever the page holds there must not reach P V.
          if (first_key + lane >= now.end || first_key + lane < now.lowest) {
            const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int v = 0; v < VALUE_CHUNKS; ++v) *reinterpret_cast<uint4*>(t + V_OFFSET + (v >> 3) * HALF_BYTES + lane * 128 + (v & 7) * 16) = zero;
          }
        }
        __syncwarp();
        if (first_key + KB - 1 > all_see || first_key < now.lowest)
          item_block<true>(qa, qs, t, t + V_OFFSET, first_key, now.lowest, last[0], last[1], c.scale_log2, st);
        else
          item_block<false>(qa, qs, t, t + V_OFFSET, first_key, now.lowest, last[0], last[1], c.scale_log2, st);
        __syncwarp();                              // every lane is done reading before the stage is refilled
        if (++stage == STAGES) { stage = 0; parity ^= 1u; }
      }
      // this stretch's part of the item
      const long long part = static_cast<long long>(worker) + now.item;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float l = st.l[half];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const int r = half * 8 + (lane >> 2);
        if (r < now.vectors) {
          float* dst = k.acc + (part * VT + r) * D + (lane & 3) * 2;
#pragma unroll
          for (int dn = 0; dn < D / 8; ++dn) *reinterpret_cast<float2*>(dst + dn * 8) = make_float2(st.o[dn][2 * half], st.o[dn][2 * half + 1]);
          if ((lane & 3) == 0) k.ml[part * VT + r] = make_float2(st.m[half], l);
        }
      }
      if (behind >= s_end) break;
      if constexpr (!kQueriesInRegisters) {
        next = locate(behind);
        fetch_queries(next);
      }
      now = next;
    }
  }
  if (k.covered > 0) pdl_wait();
}

// A vector's parts joined, a warp a vector: those of its row's item, of its group's tile, and of the tcgen05 kernel's splits.
constexpr int JOIN_WARPS = 4;
__global__ void __launch_bounds__(JOIN_WARPS * 32)
prefix_join_kernel(bf16* __restrict__ out, const StreamCall k) {
  const PrefixCall& c = k.c;
  const int lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();
  const int vec = static_cast<int>(blockIdx.x) * JOIN_WARPS + (threadIdx.x >> 5);
  if (vec >= c.n_rows * c.nh) return;
  const int group = c.nh / c.nkv;
  const int i = vec / c.nh, head = vec % c.nh, kvh = head / group;
  constexpr int PER = (D + 127) / 128;
  float4 o[PER];
#pragma unroll
  for (int n = 0; n < PER; ++n) o[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float m = -INFINITY, l = 0.0f;
  // `count` parts, `step` vectors from one to the next
  auto join = [&](const float* acc, const float2* ml, int count, int step) {
    for (int p0 = 0; p0 < count; p0 += 32) {
      float2 mine = make_float2(-INFINITY, 0.0f);
      if (p0 + lane < count) mine = __ldcg(ml + static_cast<long long>(p0 + lane) * step);
      const float most = fmaxf(m, warp_max(mine.x));
      if (most == -INFINITY) continue;
      const float f = m == -INFINITY ? 0.0f : exp2f(m - most), w = mine.x == -INFINITY ? 0.0f : exp2f(mine.x - most);
      m = most;
      l = fmaf(l, f, warp_sum(mine.y * w));
#pragma unroll
      for (int n = 0; n < PER; ++n) { o[n].x *= f; o[n].y *= f; o[n].z *= f; o[n].w *= f; }
      const int some = min(32, count - p0);
#pragma unroll 4
      for (int p = 0; p < some; ++p) {
        const float wp = __shfl_sync(0xffffffffu, w, p);
        const float* src = acc + static_cast<long long>(p0 + p) * step * D;
#pragma unroll
        for (int n = 0; n < PER; ++n) {
          const int dim = n * 128 + lane * 4;
          if ((D % 128 == 0 || dim < D) && wp > 0.0f) {      // (nothing was written where a split saw no key)
            const float4 a = __ldcg(reinterpret_cast<const float4*>(src + dim));
            o[n].x = fmaf(wp, a.x, o[n].x);
            o[n].y = fmaf(wp, a.y, o[n].y);
            o[n].z = fmaf(wp, a.z, o[n].z);
            o[n].w = fmaf(wp, a.w, o[n].w);
          }
        }
      }
    }
  };
  const Sequence& q = *k.sequence;
  const long long total = static_cast<long long>(q.blocks) * c.nkv;
  auto join_item = [&](int first, int blocks, int item, int r) {
    if (blocks <= 0) return;
    const long long s = static_cast<long long>(kvh) * q.blocks + first;
    const int w0 = worker_of(s, total, q.workers), w1 = worker_of(s + blocks - 1, total, q.workers);
    const long long part = static_cast<long long>(w0) + kvh * static_cast<long long>(q.items) + item;
    join(k.acc + (part * VT + r) * D, k.ml + part * VT + r, w1 - w0 + 1, VT);
  };
  const int e = c.n_groups + i;
  join_item(q.start[e], q.start[e + 1] - q.start[e], q.group_tiles + i, head % group);
  const int g = group_of_row(c, i);
  if (g >= 0) {
    const int2 rows = rows_of_group(c, g);
    const int v = (i - rows.x) * group + head % group;
    if (v < k.covered) {
      const long long place = static_cast<long long>(vec) * c.splits_shared;
      join(c.part_acc + place * D, c.part_ml + place, c.splits_shared, 1);
    } else {
      const int tiles = tiles_of(k, rows.y, group), tile = (v - k.covered) / VT;
      const int blocks = (q.start[g + 1] - q.start[g]) / max(tiles, 1);
      join_item(q.start[g] + tile * blocks, blocks, q.tiles_before[g] + tile, (v - k.covered) % VT);
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  bf16* dst = out + (static_cast<long long>(c.cu_q[c.rows[i]]) * c.nh + head) * D;
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    const int dim = n * 128 + lane * 4;
    if (D % 128 == 0 || dim < D) {
      const uint2 two = make_uint2(pack_bf16(o[n].x * inv, o[n].y * inv), pack_bf16(o[n].z * inv, o[n].w * inv));
      *reinterpret_cast<uint2*>(dst + dim) = two;
    }
  }
}

// Parts that the kernel may leave: one for every stretch and item.
static long long parts_of(int n_rows, int n_groups, int nh, int nkv, int sms) {
  const long long group = nh / nkv;
  return static_cast<long long>(sms) * WARPS + nkv * ((n_rows * group + VT - 1) / VT + n_groups + n_rows) + 1;
}
static long long align4(long long n) { return (n + 3) / 4 * 4; }

// Rows and groups of a call, in all.
B200_EXPORT int b200_prefix_most_entries() { return MOST_ENTRIES; }
// Floats of scratch: the tcgen05 kernel's part first (splits_shared > 0).
B200_EXPORT long long b200_prefix_scratch_floats(int n_rows, int n_groups, int nh, int nkv, int splits_shared, int sms) {
  const long long vectors = static_cast<long long>(n_rows) * nh * splits_shared, parts = parts_of(n_rows, n_groups, nh, nkv, sms) * VT;
  return vectors * (D + 2) + parts * (D + 2) + align4(sizeof(Sequence) / 4) + 8;
}

// q, out [tokens, nh * D]; k_cache, v_cache [pages, nkv, page_size, D]; `groups`: (first row, shared keys) each.  `scratch` holds
// b200_prefix_scratch_floats(...) floats on a 16-byte boundary.  `covered` > 0: b200_prefix_tcgen05 has just been launched with the
// same scratch for the first `covered` vectors of every group, in splits_shared splits (else 0 of both).  `sms`: CTAs.
B200_EXPORT int b200_prefix_attention_mma(const void* q, const void* k_cache, const void* v_cache, void* out, float* scratch, const int* block_table,
                                          int table_stride, const int* cu_q, const int* kv_len, const int* rows, int n_rows, const int* groups,
                                          int n_groups, int nh, int nkv, int page_size, int pages, float scale, int splits_shared, int covered,
                                          int sms, int* err, cudaStream_t stream) {
  if (n_rows <= 0) return 0;
  if (nh <= 0 || nkv <= 0 || nh % nkv != 0 || nh / nkv > 16 || page_size <= 0 || (page_size & (page_size - 1)) != 0 || pages <= 0 || table_stride <= 0 || n_groups < 0)
    return B200_BAD_SIZE;
  if (splits_shared < 0 || covered < 0 || (covered > 0) != (splits_shared > 0) || sms < 1 || n_rows + n_groups > MOST_ENTRIES) return B200_BAD_SIZE;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(scratch)) % 16 != 0) return B200_BAD_ALIGN;
  StreamCall k;
  const size_t vectors = static_cast<size_t>(n_rows) * nh * splits_shared, parts = static_cast<size_t>(parts_of(n_rows, n_groups, nh, nkv, sms)) * VT;
  float2* part_ml = reinterpret_cast<float2*>(scratch + vectors * D);
  k.acc = scratch + align4(vectors * (D + 2));
  k.ml = reinterpret_cast<float2*>(k.acc + parts * D);
  k.sequence = reinterpret_cast<Sequence*>(k.ml + parts);
  k.covered = covered;
  k.c = {block_table, cu_q, kv_len, rows, reinterpret_cast<const int2*>(groups), scratch, part_ml, err, table_stride, n_rows, n_groups, nh, nkv,
         page_size, pages, splits_shared, 0, 1, scale * 1.4426950408889634f};
  CUtensorMap kmap, vmap;
  const int box_rows = page_size < KB ? page_size : KB;
  const long long lines = static_cast<long long>(pages) * nkv * page_size;
  int rc = make_kv_tensor_map(&kmap, k_cache, lines, D, box_rows);
  if (rc == 0) rc = make_kv_tensor_map(&vmap, v_cache, lines, D, box_rows);
  if (rc != 0) return rc;
  static bool seen[16];
  rc = prefix_smem_limit(prefix_stream_kernel, static_cast<int>(SMEM), seen);
  if (rc != 0) return rc;
  rc = b200_launch(prefix_stream_kernel, dim3(sms), dim3(THREADS), SMEM, stream, 0, kmap, vmap, static_cast<const bf16*>(q), k, box_rows);
  if (rc != 0) return rc;
  const long long ctas = (static_cast<long long>(n_rows) * nh + JOIN_WARPS - 1) / JOIN_WARPS;
  if (ctas > INT32_MAX / JOIN_WARPS) return B200_BAD_SIZE;
  return b200_launch(prefix_join_kernel, dim3(static_cast<unsigned>(ctas)), dim3(JOIN_WARPS * 32), 0, stream, 0, static_cast<bf16*>(out), k);
}
