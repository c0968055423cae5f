// Decode attention behind shared prefixes (prefix.cuh) over the bfloat16 cache, on mma.sync.  Compile with -DHEAD_DIM=<multiple of
// 16, at most 256>; at most 16 query heads a KV head.
//
// Work comes in items: up to 16 query vectors of one KV head (a tile of a group's against its shared keys, or one row's against its
// own), an item in blocks of 32 keys.  All items' blocks stand in one sequence, and every warp of a persistent grid takes an equal
// stretch of it, whatever the rows' lengths.  A warp works alone: it fetches blocks by cp.async into a ring of its own, across the
// borders of items, multiplies them (as attention_mma.cu does) with an item's queries, which stay in registers up to 128 dims and come
// while the item before is worked on, and leaves for each item that it touches one part: float outputs, maximum, sum.  Stretch w
// and item x meet in part w + x, which rises along the sequence, so no two meet in one place and none needs to be asked for.
// A kernel behind this one joins a vector's parts.
//
// Bound, where there are many keys, by their bytes (six groups of 104 MB: 28.5 us, of which 19 at 5.5 TB/s, the rest the beginning and
// the join), else by what a warp waits for: of 2,700 cycles a block of 128 dims the products take 900, the softmax 430, asking for the next
// block 800.  (That by the copy engine, a box of 64 dims of a page a copy: 900, with a wait for the page's number in front 1,400, and the
// calls 1 to 2.5 us slower; a box of all dims a copy: 500, with a longer way until the first one is there, 8.5 us for 8.3 at two rows
// behind 300 keys, 21.3 for 19.9 at four groups of eight behind 1,000, 73.9 for 75.3 at 64 behind 32,768.  A CTA an item with a split,
// warps joined in shared memory: 64 rows of 1 to 1,024 own keys, 8 KV heads, 52 us, most of it the CTAs' beginnings and ends.)  A group
// of more than 16 vectors reads its shared keys once for each 16 (from the second-level cache), which prefix_tcgen05.cu does not.
#include "attention_mma.cuh"
#include "prefix.cuh"

constexpr bool kQueriesInRegisters = D <= 128;
constexpr int VT = 16;                           // query vectors of an item
constexpr int STAGES = 2;
constexpr int WARPS = D <= 64 ? 8 : D <= 128 ? 6 : D <= 192 ? 4 : 3;
constexpr int THREADS = WARPS * 32;
constexpr int MOST_ENTRIES = 400;                // rows and groups of a call, whose places in the sequence stand in shared memory
constexpr size_t RING = static_cast<size_t>(WARPS) * STAGES * TILE_BYTES;
constexpr size_t QUERIES = static_cast<size_t>(WARPS) * VT * LD * sizeof(bf16);
constexpr size_t FIXED = 128 + RING + QUERIES;

// The places of a call's groups, then rows, in the sequence of blocks (of one KV head), in shared memory.
struct Entries {
  int* start;                                    // [entries + 1]: the first block
  int* keys;                                     // a group's shared keys, a row's keys
  int* low;                                      // a group's first row; a row's first own key
  int* where;                                    // the tiles of the groups before; a row's place in the block table
  int* token;                                    // a row's token
  int blocks, items, group_tiles;                // in all (of one KV head)
};
__host__ __device__ constexpr int entries_bytes(int n_entries) { return (5 * n_entries + 1 + 8) * 4; }
static_assert(WARPS <= 8, "a sum a warp");
static_assert(FIXED + entries_bytes(MOST_ENTRIES) <= 227 * 1024, "shared memory of one CTA");

// Which parts make up a row's vectors of one KV head: those of its own item, and of the tiles of its group that the vectors are in (at
// most two, `first_vector` counted from the first vector behind those that the tcgen05 kernel serves).
struct __align__(16) RowParts { int own, own_count, first_vector, tile[2], tile_count[2], grouped; };

struct StreamCall {
  PrefixCall c;                                  // part_acc, part_ml: of the tcgen05 kernel, [n_rows * nh][splits_shared]
  float* acc;                                    // [parts][16][D]
  float2* ml;                                    // [parts][16]
  RowParts* row_parts;                           // [n_rows][nkv]
  int covered, covered_groups;                   // vectors of each of the first groups that the tcgen05 kernel serves, and how many groups
  __device__ __forceinline__ int covered_of(int g) const { return g < covered_groups ? covered : 0; }
};

__device__ __forceinline__ int tiles_of(const StreamCall& k, int g, int rows, int group) { return (max(0, rows * group - k.covered_of(g)) + VT - 1) / VT; }

// Sums of `v` over the CTA's threads before this one; `sum` becomes that of all.  `sh`: one int a warp.
template <int WARPS_HERE>
__device__ __forceinline__ int sums_before(int v, int& sum, int* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int upto = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int less = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += less;
  }
  if (lane == 31) sh[warp] = upto;
  __syncthreads();
  int before = 0;
  sum = 0;
#pragma unroll
  for (int w = 0; w < WARPS_HERE; ++w) {
    if (w == warp) before = sum;
    sum += sh[w];
  }
  __syncthreads();
  return before + upto - v;
}

// The group of the i-th row, the last one that begins at or before it (-1: none does).
__device__ __forceinline__ int group_of(const Entries& at, int n_groups, int i) {
  int lo = 0, hi = n_groups;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (at.low[mid] <= i) lo = mid + 1; else hi = mid;
  }
  return lo - 1;
}

// Fills in `at` (a whole CTA).  What the kernels wait for here is two loads one behind the other, a row's number and its length.
template <int WARPS_HERE>
__device__ __forceinline__ void lay_out(const StreamCall& k, Entries& at, int* memory) {
  constexpr int N = WARPS_HERE * 32;
  const PrefixCall& c = k.c;
  const int n_entries = c.n_groups + c.n_rows, group = c.nh / c.nkv;
  at.start = memory;
  at.keys = at.start + n_entries + 1;
  at.low = at.keys + n_entries;
  at.where = at.low + n_entries;
  at.token = at.where + n_entries;
  int* sh = at.token + n_entries;
  const int most = static_cast<int>(min(static_cast<long long>(c.table_stride) * c.page_size, static_cast<long long>(INT_MAX)));
  auto checked = [&](int keys) {                   // no more keys than a block table has places for
    if (keys > most) atomicOr(c.err, B200_ERR_SLOT_RANGE);
    return min(max(keys, 0), most);
  };
  for (int x = threadIdx.x; x < max(c.n_groups, c.n_rows); x += N) {
    const bool is_row = x < c.n_rows, is_group = x < c.n_groups;
    const int row = is_row ? c.rows[x] : 0;
    const int2 here = is_group ? c.groups[x] : make_int2(0, 0);
    const int behind = is_group && x + 1 < c.n_groups ? c.groups[x + 1].x : c.n_rows;
    const int keys = is_row ? c.kv_len[row] : 0, token = is_row ? c.cu_q[row] : 0;
    if (is_group) {
      const int first = min(max(here.x, 0), c.n_rows), rows = min(max(behind, first), c.n_rows) - first;
      at.keys[x] = rows > 0 ? checked(here.y) : 0;
      at.low[x] = first;
      at.where[x] = tiles_of(k, x, rows, group);
    }
    if (is_row) {
      at.where[c.n_groups + x] = row;
      at.keys[c.n_groups + x] = checked(keys);
      at.token[c.n_groups + x] = token;
    }
  }
  __syncthreads();
  at.blocks = at.group_tiles = 0;
  for (int e0 = 0; e0 < n_entries; e0 += N) {
    const int e = e0 + static_cast<int>(threadIdx.x);
    int v = 0, tiles = 0;
    if (e < c.n_groups) {
      tiles = at.where[e];
      v = tiles * ((at.keys[e] + KB - 1) / KB);
    } else if (e < n_entries) {
      const int g = group_of(at, c.n_groups, e - c.n_groups);
      const int keys = at.keys[e], low = g < 0 ? 0 : min(keys, at.keys[g]);
      at.low[e] = low;
      v = keys > low ? (keys + KB - 1) / KB - low / KB : 0;
    }
    int sum, before = sums_before<WARPS_HERE>(v, sum, sh);
    if (e < n_entries) at.start[e] = at.blocks + before;
    at.blocks += sum;
    if (e0 < c.n_groups) {
      before = sums_before<WARPS_HERE>(tiles, sum, sh);
      if (e < c.n_groups) at.where[e] = at.group_tiles + before;
      at.group_tiles += sum;
    }
  }
  if (threadIdx.x == 0) at.start[n_entries] = at.blocks;
  at.items = at.group_tiles + c.n_rows;
  __syncthreads();
}

// The sequence of all KV heads' blocks in equal stretches, the last one what is left: as many blocks as the longest has to have anyway, for
// every stretch costs a part more.  (Stretches that differ by a block, on all workers: eight rows behind 4,096 keys 16.1 us, 15.0 so.)
struct Stretches {
  int blocks, workers;
  __device__ __forceinline__ Stretches(int total, int most) : blocks(max(1, (total + most - 1) / most)), workers((total + blocks - 1) / blocks), total_(total) {}
  __device__ __forceinline__ int begin(int w) const { return min(w * blocks, total_); }
  __device__ __forceinline__ int of(int s) const { return s / blocks; }
 private:
  int total_;
};

// Where a worker stands: `left` blocks of an item from key first_key on.
struct Place {
  int s, kvh, first_key, end, lowest, left, item, i0, vector0, vectors, table_row;
};
// (not inlined: it is asked in three places, and a kernel this short waits for its instructions)
__device__ __noinline__ Place locate(const Entries& at, int s, int s_end, int n_groups, int n_rows, int group, int covered, int covered_groups) {
  Place p;
  p.s = s;
  p.kvh = s / at.blocks;
  const int pos = s - p.kvh * at.blocks, lane = threadIdx.x & 31;
  int e = -1;                                      // the entries that begin at or before pos: the last of them holds it
  for (int e0 = 0; e0 < n_groups + n_rows; e0 += 32) {
    const unsigned begun = __ballot_sync(0xffffffffu, e0 + lane < n_groups + n_rows && at.start[e0 + lane] <= pos);
    e += __popc(begun);
    if (begun != 0xffffffffu) break;
  }
  int block = pos - at.start[e], of;
  p.end = at.keys[e];
  if (e < n_groups) {
    of = (p.end + KB - 1) / KB;
    const int tile = block / of;
    block -= tile * of;
    p.item = p.kvh * at.items + at.where[e] + tile;
    p.lowest = 0;
    p.i0 = at.low[e];
    const int next = e + 1 < n_groups ? max(at.low[e + 1], p.i0) : n_rows;
    p.vector0 = (e < covered_groups ? covered : 0) + tile * VT;
    p.vectors = min(VT, (next - p.i0) * group - p.vector0);
    p.table_row = at.where[n_groups + p.i0];
    p.first_key = block * KB;
  } else {
    p.lowest = at.low[e];
    of = (p.end + KB - 1) / KB - p.lowest / KB;
    p.i0 = e - n_groups;
    p.item = p.kvh * at.items + at.group_tiles + p.i0;
    p.vector0 = 0;
    p.vectors = group;
    p.table_row = at.where[e];
    p.first_key = (p.lowest / KB + block) * KB;
  }
  p.left = min(of - block, s_end - s);
  return p;
}

// What the block table says of the page of this lane's keys, asked for a block before it is used: a block is cut into boxes, the keys of
// one page each, and lane j has the j-th; pages of no power of two end anywhere in a block, and a box is a key then (log2_page -1).  A
// box that ends below `lowest` is another table's: the sink's page, 0, and so is what a lane without a box gets.
struct Boxes { int log2_rows, log2_page; };
__device__ __forceinline__ int page_of_key(const PrefixCall& c, const Boxes& boxes, int key) {
  return boxes.log2_page >= 0 ? key >> boxes.log2_page : key / c.page_size;
}
__device__ __forceinline__ int lane_page(const PrefixCall& c, const Boxes& boxes, const Place& p, int lane) {
  const int key0 = p.first_key + (lane << boxes.log2_rows);
  if ((lane << boxes.log2_rows) >= KB || key0 >= p.end || key0 + (1 << boxes.log2_rows) <= p.lowest) return 0;
  return __ldg(c.block_table + static_cast<long long>(p.table_row) * c.table_stride + page_of_key(c, boxes, key0));
}
// The warp asks for the block at p.first_key, its boxes on the lanes' pages (the sink's for one outside the pool); rows that are not the
// item's become zeros, so that whatever a page holds there does not reach P V.
__device__ __forceinline__ void fetch_block_of(const PrefixCall& c, const Boxes& boxes, const Place& p, int page, const bf16* __restrict__ kc,
                                               const bf16* __restrict__ vc, unsigned char* tile, int lane) {
  constexpr int CHUNKS = D / 8, TURNS = KB * CHUNKS / 32, ROWS = 32 / CHUNKS;      // of 16 bytes in a row; rows a turn of the warp's lanes
  if (page < 0 || page >= c.pages) {
    atomicOr(c.err, B200_ERR_SLOT_RANGE);
    page = 0;
  }
  const int key0 = p.first_key + (lane << boxes.log2_rows);
  const int y = (page * c.nkv + p.kvh) * c.page_size + key0 - page_of_key(c, boxes, key0) * c.page_size;
  const int from = p.lowest - p.first_key, to = p.end - p.first_key;
  if (32 % CHUNKS == 0 && ROWS <= 8 && boxes.log2_rows >= 3) {      // eight keys behind one another at a time
#pragma unroll
    for (int r8 = 0; r8 < KB; r8 += 8) {
      const int mine = lane / CHUNKS, chunk = lane % CHUNKS;
      const int line = __shfl_sync(0xffffffffu, y, r8 >> boxes.log2_rows) + (r8 & ((1 << boxes.log2_rows) - 1)) + mine;
      const long long at = static_cast<long long>(line) * D + chunk * 8;
#pragma unroll
      for (int r = 0; r < 8; r += ROWS <= 8 ? ROWS : 8) {
        const int row = r8 + r + mine;
        unsigned char* dst = tile + swz(row, chunk);
        cp_async16(dst, kc + at + r * D, row >= from && row < to);
        cp_async16(dst + V_OFFSET, vc + at + r * D, row >= from && row < to);
      }
    }
    return;
  }
#pragma unroll
  for (int x = 0; x < TURNS; ++x) {
    const int row = (x * 32 + lane) / CHUNKS, chunk = (x * 32 + lane) % CHUNKS;
    const int line = __shfl_sync(0xffffffffu, y, row >> boxes.log2_rows) + (row & ((1 << boxes.log2_rows) - 1));
    const long long at = static_cast<long long>(line) * D + chunk * 8;
    unsigned char* dst = tile + swz(row, chunk);
    cp_async16(dst, kc + at, row >= from && row < to);
    cp_async16(dst + V_OFFSET, vc + at, row >= from && row < to);
  }
}

// One block of 32 keys against the 16 vectors whose queries are `qa` (or stand at `qs`): as block_mma of attention_mma.cuh, with the
// last key that a vector sees (last0, last1: of rows lane / 4 and lane / 4 + 8; -1: none) and the item's first.
__device__ __forceinline__ void item_block(const uint32_t (&qa)[kQueriesInRegisters ? D / 16 : 1][4], const bf16* qs, const unsigned char* ks,
                                           const unsigned char* vs, bool masked, int first_key, int lowest, int last0, int last1, float scale_log2,
                                           WarpAcc& st) {
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
  if (masked) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int key = first_key + n * 8 + t2 + e;
        s[n][e] = key >= lowest && key <= last0 ? s[n][e] : -INFINITY;
        s[n][2 + e] = key >= lowest && key <= last1 ? s[n][2 + e] : -INFINITY;
      }
    }
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    mx0 = fmaxf(mx0, fmaxf(s[n][0], s[n][1]));
    mx1 = fmaxf(mx1, fmaxf(s[n][2], s[n][3]));
  }
  mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1)); mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
  mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1)); mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
  const float m0 = fmaxf(st.m[0], mx0 * scale_log2), m1 = fmaxf(st.m[1], mx1 * scale_log2);      // (the scale is positive)
  const float base0 = m0 == -INFINITY ? 0.0f : m0, base1 = m1 == -INFINITY ? 0.0f : m1;
  const float c0 = fast_exp2(st.m[0] - base0), c1 = fast_exp2(st.m[1] - base1);       // (0 on the first visible block)
  float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      s[n][e] = fast_exp2(fmaf(s[n][e], scale_log2, -base0));
      s[n][2 + e] = fast_exp2(fmaf(s[n][2 + e], scale_log2, -base1));
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
prefix_stream_kernel(const bf16* __restrict__ kc, const bf16* __restrict__ vc, const bf16* __restrict__ q,
                     const StreamCall k, const Boxes boxes) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  bf16* queries = reinterpret_cast<bf16*>(tiles + RING);
  const PrefixCall& c = k.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // Behind the tcgen05 kernel of the same call, which has waited for the kernels before it, this one begins beside it, and waits
  // for its end at its own: whoever waits for this kernel then waits for both.  The joining kernel may come as soon as what was
  // launched before the call has ended.
  if (threadIdx.x < 32) prefetch_indices(c);
  if (k.covered == 0) pdl_wait();
  pdl_launch_dependents();
  Entries at;
  lay_out<WARPS>(k, at, reinterpret_cast<int*>(reinterpret_cast<unsigned char*>(queries) + QUERIES));

  const int group = c.nh / c.nkv;
  const Stretches stretches(at.blocks * c.nkv, static_cast<int>(gridDim.x) * WARPS);
  const int worker = warp * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x);      // (few stretches: on as many SMs as can be)
  const int s_begin = worker < stretches.workers ? stretches.begin(worker) : 0, s_end = worker < stretches.workers ? stretches.begin(worker + 1) : 0;
  if (s_begin < s_end) {
    unsigned char* ring = tiles + static_cast<size_t>(warp) * STAGES * TILE_BYTES;
    bf16* qs = queries + warp * VT * LD;
    // the queries of an item into shared memory: two lanes a vector
    auto fetch_queries = [&](const Place& p) {
      const int r = lane >> 1, vec = p.vector0 + min(r, p.vectors - 1), row = vec / group;
      const int token = at.token[c.n_groups + p.i0 + row];
      const bf16* src = q + (static_cast<long long>(token) * c.nh + p.kvh * group + vec - row * group) * D;
      for (int part = lane & 1; part < D / 8; part += 2) cp_async16(qs + r * LD + part * 8, src + part * 8, r < p.vectors);
      cp_async_commit();
    };
    Place now = locate(at, s_begin, s_end, c.n_groups, c.n_rows, group, k.covered, k.covered_groups), ahead = now, next = now;
    int page = lane_page(c, boxes, ahead, lane);
    fetch_queries(now);
    uint32_t qa[kQueriesInRegisters ? D / 16 : 1][4];
    WarpAcc st;
    int last[2], all_see = 0, done = 0;            // `done`: blocks of the item behind us
    int fetch_stage = 0, stage = 0;
    for (int tick = 1 - STAGES;; ++tick) {
      // the next block of the stretch on its way, whatever item it is of; the page numbers of the one behind it are asked for
      if (ahead.s < s_end) {
        fetch_block_of(c, boxes, ahead, page, kc, vc, ring + fetch_stage * TILE_BYTES, lane);
        fetch_stage = fetch_stage + 1 == STAGES ? 0 : fetch_stage + 1;
        ++ahead.s;
        ahead.first_key += KB;
        if (--ahead.left == 0 && ahead.s < s_end) ahead = locate(at, ahead.s, s_end, c.n_groups, c.n_rows, group, k.covered, k.covered_groups);
        if (ahead.s < s_end) page = lane_page(c, boxes, ahead, lane);
      }
      cp_async_commit();                           // (one a tick; an item's queries are one more, behind that of a tick)
      if (tick < 0) continue;
      if (done == 0) {                             // an item begins
        cp_async_wait<1>();
        __syncwarp();
        if constexpr (kQueriesInRegisters) {
#pragma unroll
          for (int x = 0; x < D / 16; ++x) ldmatrix_x4(qa[x], qs + (lane & 15) * LD + x * 16 + (lane >> 4) * 8);
          __syncwarp();
          if (now.s + now.left < s_end) {
            next = locate(at, now.s + now.left, s_end, c.n_groups, c.n_rows, group, k.covered, k.covered_groups);
            fetch_queries(next);
          }
        }
        // the last key that this lane's two vectors see, and the least of all vectors'
        all_see = INT_MAX;
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
        st.init();
      }
      cp_async_wait<STAGES - 1>();
      __syncwarp();
      unsigned char* t = ring + stage * TILE_BYTES;
      const int first_key = now.first_key + done * KB;
      item_block(qa, qs, t, t + V_OFFSET, first_key + KB - 1 > all_see || first_key < now.lowest, first_key, now.lowest, last[0], last[1], c.scale_log2, st);
      __syncwarp();                                // every lane is done reading before the stage is refilled
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      if (++done < now.left) continue;
      // the item ends here, or the stretch: its part
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
          if ((lane & 3) == 0) k.ml[part * VT + r] = part_of(st.m[half], l);
        }
      }
      if (now.s + now.left >= s_end) break;
      if constexpr (!kQueriesInRegisters) {
        next = locate(at, now.s + now.left, s_end, c.n_groups, c.n_rows, group, k.covered, k.covered_groups);
        fetch_queries(next);
      }
      now = next;
      done = 0;
    }
  }
  // what the joining kernel goes by
  for (int x = static_cast<int>(threadIdx.x) * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x); x < c.n_rows * c.nkv; x += static_cast<int>(gridDim.x) * THREADS) {
    const int i = x / c.nkv, kvh = x - i * c.nkv, e = c.n_groups + i;
    auto parts_of_item = [&](int first, int blocks, int item, int& part) {      // of a run of blocks: the number of parts, the first
      part = 0;
      if (blocks <= 0) return 0;
      const int s = kvh * at.blocks + first, w0 = stretches.of(s);
      part = w0 + kvh * at.items + item;
      return stretches.of(s + blocks - 1) - w0 + 1;
    };
    RowParts p = {};
    p.own_count = parts_of_item(at.start[e], at.start[e + 1] - at.start[e], at.group_tiles + i, p.own);
    const int g = group_of(at, c.n_groups, i);
    p.grouped = g >= 0;
    if (g >= 0) {
      p.first_vector = (i - at.low[g]) * group - k.covered_of(g);
      const int tiles_here = (g + 1 < c.n_groups ? at.where[g + 1] : at.group_tiles) - at.where[g];
      const int blocks_here = tiles_here > 0 ? (at.start[g + 1] - at.start[g]) / tiles_here : 0, tile = max(p.first_vector, 0) / VT;
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (tile + t < tiles_here) p.tile_count[t] = parts_of_item(at.start[g] + (tile + t) * blocks_here, blocks_here, at.where[g] + tile + t, p.tile[t]);
    }
    k.row_parts[x] = p;
  }
  if (k.covered > 0) pdl_wait();
}

// A vector joined out of its parts: those of its group's tile, or of the tcgen05 kernel's splits, and those of its row's item.  grid (n_rows
// * nh).  (A CTA four vectors, two warps each, weights before outputs: eight rows behind 4,096 keys 12,800 cycles.)
template <int JOIN_WARPS>
__global__ void __launch_bounds__(JOIN_WARPS * 32)
prefix_join_kernel(bf16* __restrict__ out, const StreamCall k) {
  __shared__ __align__(16) JoinShared<D, JOIN_WARPS> left;
  const PrefixCall& c = k.c;
  const int group = c.nh / c.nkv;
  const int i = static_cast<int>(blockIdx.x) / c.nh, head = static_cast<int>(blockIdx.x) - i * c.nh, kvh = head / group, r = head - kvh * group;
  // (the stream kernel began when everything before the call had ended, so the call's index arrays may be read beside it)
  bf16* dst = out + (static_cast<long long>(c.cu_q[c.rows[i]]) * c.nh + head) * D;
  pdl_launch_dependents();
  pdl_wait();
  const RowParts* row = k.row_parts + static_cast<long long>(i) * c.nkv + kvh;
  const int4 first = *reinterpret_cast<const int4*>(row), rest = *(reinterpret_cast<const int4*>(row) + 1);
  const int own = first.x, own_count = first.y, v = first.z + r, grouped = rest.w;
  const bool second = v / VT > max(first.z, 0) / VT, split = grouped != 0 && v < 0;
  const int tile = second ? rest.x : first.w;
  const int tile_count = grouped == 0 ? 0 : split ? c.splits_shared : second ? rest.z : rest.y;
  const long long vec = static_cast<long long>(blockIdx.x) * c.splits_shared;
  join_parts<D, JOIN_WARPS>(dst, D, tile_count + own_count, [&](int p, const float2*& ml, const float*& acc) {
    const bool of_tc = split && p < tile_count;
    const long long at = of_tc ? vec + p : p < tile_count ? static_cast<long long>(tile + p) * VT + v % VT : static_cast<long long>(own + p - tile_count) * VT + r;
    ml = (of_tc ? c.part_ml : k.ml) + at;
    acc = (of_tc ? c.part_acc : k.acc) + at * D;
  }, left);
}

// Parts that the kernel may leave: one for every stretch and item.
static long long parts_of(int n_rows, int n_groups, int nh, int nkv, int ctas) {
  const long long group = nh / nkv;
  return static_cast<long long>(ctas) * WARPS + nkv * ((n_rows * group + VT - 1) / VT + n_groups + n_rows) + 1;
}
static long long align4(long long n) { return (n + 3) / 4 * 4; }

// Floats of scratch: the tcgen05 kernel's part first (splits_shared > 0).
B200_EXPORT long long b200_prefix_scratch_floats(int n_rows, int n_groups, int nh, int nkv, int splits_shared, int ctas) {
  const long long vectors = static_cast<long long>(n_rows) * nh * splits_shared, parts = parts_of(n_rows, n_groups, nh, nkv, ctas) * VT;
  return align4(vectors * (D + 2)) + parts * (D + 2) + static_cast<long long>(n_rows) * nkv * (sizeof(RowParts) / 4);
}

// q, out [tokens, nh * D]; k_cache, v_cache [pages, nkv, page_size, D]; `groups`: (first row, shared keys) each.  `scratch` holds
// b200_prefix_scratch_floats(...) floats on a 16-byte boundary (of as many `ctas`).  `covered` > 0: b200_prefix_tcgen05 has just been launched with the
// same scratch for the first covered % 2^16 vectors of every one of the first covered / 2^16 groups (0: of all), in splits_shared splits (else 0 of
// both).  `ctas`: of the stream kernel, at most one for each of the device's `sms`.
B200_EXPORT int b200_prefix_attention_mma(const void* q, const void* k_cache, const void* v_cache, void* out, float* scratch, const int* block_table,
                                          int table_stride, const int* cu_q, const int* kv_len, const int* rows, int n_rows, const int* groups,
                                          int n_groups, int nh, int nkv, int page_size, int pages, float scale, int splits_shared, int covered,
                                          int ctas, int sms, int* err, cudaStream_t stream) {
  if (n_rows <= 0) return 0;
  if (nh <= 0 || nkv <= 0 || nh % nkv != 0 || nh / nkv > 16 || page_size <= 0 || pages <= 0 || table_stride <= 0 || n_groups < 0)
    return B200_BAD_SIZE;
  // (blocks are counted in 32 bits)
  const long long most_blocks = (static_cast<long long>(table_stride) * page_size / KB + 2) * nkv *
                                ((static_cast<long long>(n_rows) * (nh / nkv) + VT - 1) / VT + n_groups + n_rows);
  if (most_blocks > INT32_MAX / 2) return B200_BAD_SIZE;
  if (splits_shared < 0 || covered < 0 || (covered > 0) != (splits_shared > 0) || ctas < 1 || ctas > sms || n_rows + n_groups > MOST_ENTRIES) return B200_BAD_SIZE;
  if (!prefix_can_be_served({q, k_cache, v_cache, out, scratch, block_table, cu_q, kv_len, rows, err}, groups, n_groups, table_stride, page_size))
    return B200_BAD_SIZE;
  if (static_cast<long long>(pages) * nkv * page_size > INT32_MAX) return B200_BAD_SIZE;      // (a copy's row is counted in 32 bits)
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(scratch)) % 16 != 0) return B200_BAD_ALIGN;
  StreamCall k;
  const size_t vectors = static_cast<size_t>(n_rows) * nh * splits_shared, parts = static_cast<size_t>(parts_of(n_rows, n_groups, nh, nkv, ctas)) * VT;
  if (static_cast<long long>(n_rows) * nh > INT32_MAX) return B200_BAD_SIZE;
  float2* part_ml = reinterpret_cast<float2*>(scratch + vectors * D);
  k.acc = scratch + align4(vectors * (D + 2));
  k.ml = reinterpret_cast<float2*>(k.acc + parts * D);
  k.row_parts = reinterpret_cast<RowParts*>(k.ml + parts);
  k.covered = covered & 0xffff;
  k.covered_groups = covered >> 16 == 0 ? n_groups : covered >> 16;
  k.c = {block_table, cu_q, kv_len, rows, reinterpret_cast<const int2*>(groups), scratch, part_ml, err, table_stride, n_rows, n_groups, nh, nkv,
         page_size, pages, splits_shared, 0, 1, scale * 1.4426950408889634f};
  Boxes boxes;
  boxes.log2_page = (page_size & (page_size - 1)) != 0 ? -1 : __builtin_ctz(page_size);
  boxes.log2_rows = boxes.log2_page < 0 ? 0 : page_size < KB ? boxes.log2_page : __builtin_ctz(KB);
  static bool seen[16];
  int rc = prefix_smem_limit(prefix_stream_kernel, static_cast<int>(FIXED) + entries_bytes(MOST_ENTRIES), seen);
  if (rc != 0) return rc;
  const int entries = entries_bytes(n_rows + n_groups);
  rc = b200_launch(prefix_stream_kernel, dim3(ctas), dim3(THREADS), FIXED + entries, stream, 0, static_cast<const bf16*>(k_cache), static_cast<const bf16*>(v_cache), static_cast<const bf16*>(q), k, boxes);
  if (rc != 0) return rc;
  const int warps = join_warps_of(static_cast<long long>(n_rows) * nh, sms);
  return b200_launch(warps == 16 ? prefix_join_kernel<16> : warps == 8 ? prefix_join_kernel<8> : warps == 4 ? prefix_join_kernel<4> : prefix_join_kernel<2>, dim3(static_cast<unsigned>(n_rows) * nh),
                     dim3(warps * 32), 0, stream, 0, static_cast<bf16*>(out), k);
}
