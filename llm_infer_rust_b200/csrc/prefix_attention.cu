// Decode attention behind shared prefixes (prefix.cuh) for float32, and for what the bfloat16 kernels do not take (head sizes that are
// no multiple of 16 or above 256, more than 16 query heads a KV head, more than 400 rows and groups, tensors off 16 bytes, tables and
// caches that they cannot count).  Compile with -DHEAD_DIM=<multiple of 16, at most 512>; the real head size may be smaller.
//
// A CTA has a tile of up to 32 query vectors and walks its split of the keys in blocks of 32, two blocks of keys and values on their
// way where they fit.  S = Q K^T (a warp eight keys) and O += P V (a warp every fourth group of eight dims) run on mma.sync in
// TF32, each float as the sum of two: x = h + l, h = x rounded to 11 bits, l = x - h cut off at as many, and x y = h h + h l + l h up to
// 2^-22 |x y| (bfloat16 keys and values are their own h).  A key of 128 dims against 32 vectors is 98 thousand products of which a multiprocessor's
// FMA units do 128 a cycle; fed from shared memory they did a third of that, for a read of 16 bytes a lane takes four cycles whether the lanes'
// places differ or not.
// Two terms do not make up an infinity, nor a float that rounding to 11 bits carries beyond the largest, nor one whose second term falls below the
// smallest.  What comes of the first two in a score or a value is never finite and stays so to the end; of the third come outputs below
// 2^-80.  The kernel that joins the splits does such a vector again, in FMA (attend_again).  (The same at the end of the kernel that attends: 19.0
// us for 17.9 at 13 rows behind 1,501 keys of 96, 154.7 for 142.5 at 48 behind 4,000 with 600 of their own.)
#include "prefix.cuh"

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<head size, a multiple of 16>"
#endif
static_assert(HEAD_DIM % 16 == 0 && HEAD_DIM >= 16 && HEAD_DIM <= 512, "head sizes 16 to 512 in steps of 16");

constexpr int D = HEAD_DIM;
constexpr int VT = 32, KB = 32, THREADS = 128;
// Padded rows: lane (g, t) of a fragment reads row g, column t of keys, queries and weights (rows 4 or 20 banks apart) or row t, column g of
// values (8 or 24 apart), and no two in one bank.
constexpr int LD = D + 4, LDV = D + 8, LDP = KB + 4;
constexpr int TILE = KB * (LD + LDV);           // floats of a block's keys and values
constexpr int FIXED = VT * LD + VT * LDP + 4 * VT;
constexpr int NT = (D / 8 + 3) / 4;             // groups of eight dims of a warp
constexpr int STAGES = (FIXED + 2 * TILE) * 4 <= 220 * 1024 ? 2 : 1;
constexpr int SMEM = (FIXED + STAGES * TILE) * 4;
static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");

// Rows first_key .. first_key + 31 of one KV head into `k` and `v` (zeros from `end` on).  Four threads a key.
template <typename T>
__device__ __forceinline__ void load_block(float* k, float* v, const T* __restrict__ kc, const T* __restrict__ vc, const PrefixCall& c,
                                           const PrefixItem& it, int first_key, int hd, bool wide) {
  const int j = threadIdx.x >> 2, part = threadIdx.x & 3;
  const int key = first_key + j;
  bool valid = key < it.end;
  long long row = 0;
  if (valid) {
    const int page = it.table[key / c.page_size];
    if (page < 0 || page >= c.pages) {
      atomicOr(c.err, B200_ERR_SLOT_RANGE);
      valid = false;
    } else {
      row = ((static_cast<long long>(page) * c.nkv + it.kvh) * c.page_size + key % c.page_size) * hd;
    }
  }
  float* kd = k + j * LD;
  float* vd = v + j * LDV;
  if constexpr (sizeof(T) == 4) {
    if (wide) {
      for (int col = part; col < hd / 4; col += 4) {
        cp_async16(kd + col * 4, kc + row + col * 4, valid);
        cp_async16(vd + col * 4, vc + row + col * 4, valid);
      }
      return;
    }
  }
  for (int pair = part; pair < hd / 2; pair += 4) {
    float2 a = make_float2(0.0f, 0.0f), b = a;
    if (valid) {
      a = make_float2(to_f32<T>(kc[row + 2 * pair]), to_f32<T>(kc[row + 2 * pair + 1]));
      b = make_float2(to_f32<T>(vc[row + 2 * pair]), to_f32<T>(vc[row + 2 * pair + 1]));
    }
    *reinterpret_cast<float2*>(kd + 2 * pair) = a;
    *reinterpret_cast<float2*>(vd + 2 * pair) = b;
  }
}

// The queries of up to `most` vectors into `qs`, scaled (zeros for those that are none and for padded columns), and the padded columns of
// keys and values, which stay zeros.  Lane r of every warp gets the first key that is not vector r's.
template <typename T>
__device__ __forceinline__ int load_queries(const T* __restrict__ q, const PrefixCall& c, const PrefixItem& it, int hd, int most, int row, float* qs, float* tiles) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = c.nh / c.nkv;
  // lane r finds vector r's place (`row`: its batch row), and four vectors' loads are on their way at once (one after the other they took
  // 10,000 cycles)
  long long mine = -1;
  int limit = 0;
  if (row >= 0) {
    const int token = c.cu_q[row];
    limit = min(it.end, keys_of_row(c, row));
    mine = (static_cast<long long>(token) * c.nh + it.kvh * group + (it.vector0 + lane) % group) * hd;
  }
  constexpr int PER = (D + 31) / 32, TURN = PER <= 4 ? 4 : 2;
  for (int r0 = warp * TURN; r0 < most; r0 += THREADS / 32 * TURN) {
    T x[TURN][PER];
#pragma unroll
    for (int y = 0; y < TURN; ++y) {
      const long long at = __shfl_sync(0xffffffffu, mine, r0 + y);
#pragma unroll
      for (int n = 0; n < PER; ++n) {
        x[y][n] = from_f32<T>(0.0f);
        if (at >= 0 && lane + 32 * n < hd) x[y][n] = q[at + lane + 32 * n];
      }
    }
#pragma unroll
    for (int y = 0; y < TURN; ++y)
#pragma unroll
      for (int n = 0; n < PER; ++n)
        if (D % 32 == 0 || lane + 32 * n < D) qs[(r0 + y) * LD + lane + 32 * n] = to_f32<T>(x[y][n]) * c.scale_log2;
  }
  if (hd < D)
    for (int i = threadIdx.x; i < STAGES * KB * (D - hd); i += THREADS) {
      const int line = i / (D - hd), dim = hd + i % (D - hd);
      float* tile = tiles + line / KB * TILE;
      tile[line % KB * LD + dim] = tile[KB * LD + line % KB * LDV + dim] = 0.0f;
    }
  return limit;
}

// x = h + l in TF32.
__device__ __forceinline__ void two_terms(float x, uint32_t& h, uint32_t& l) {
  asm("cvt.rna.tf32.f32 %0, %1;\n" : "=r"(h) : "f"(x));
  l = __float_as_uint(x - __uint_as_float(h));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 rows x 8 columns at `p` (rows `ld` apart) as the A operand.
__device__ __forceinline__ void load_a(const float* p, int ld, uint32_t (&h)[4], uint32_t (&l)[4]) {
  const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
  two_terms(p[g * ld + t], h[0], l[0]);
  two_terms(p[(g + 8) * ld + t], h[1], l[1]);
  two_terms(p[g * ld + t + 4], h[2], l[2]);
  two_terms(p[(g + 8) * ld + t + 4], h[3], l[3]);
}
// a b, a and b in two terms: the first terms' product to `large`, the others' to `small`; EXACT: b is its first term.  The tensor cores cut
// their sums off where they add to an accumulator, always towards zero: what goes into one is a few of them (all products of a split in
// one: 1.5e-6 of the result, all of it below), and longer sums are FMA units'.
template <bool EXACT>
__device__ __forceinline__ void product(float (&large)[4], float (&small)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], float b0, float b1) {
  if constexpr (EXACT) {
    mma_tf32(small, al, __float_as_uint(b0), __float_as_uint(b1));
    mma_tf32(large, ah, __float_as_uint(b0), __float_as_uint(b1));
  } else {
    uint32_t h0, l0, h1, l1;
    two_terms(b0, h0, l0);
    two_terms(b1, h1, l1);
    mma_tf32(small, al, h0, h1);
    mma_tf32(small, ah, l0, l1);
    mma_tf32(large, ah, h0, h1);
  }
}

// Where vector r's results of this split go.
__device__ __forceinline__ long long place_of(const PrefixCall& c, const PrefixItem& it, int r) {
  const int group = c.nh / c.nkv, vec = it.vector0 + r;
  return (static_cast<long long>(it.i0 + vec / group) * c.nh + it.kvh * group + vec % group) * prefix_splits(c) + it.slot;
}

// Up to 16 MT vectors against the item's keys; the results go to the vectors' slots.
template <typename T, int MT>
__device__ __forceinline__ void attend(const T* __restrict__ q, const T* __restrict__ kc, const T* __restrict__ vc, const PrefixCall& c,
                                       const PrefixItem& it, int hd, bool wide, float* sm) {
  constexpr bool EXACT = sizeof(T) == 2;
  float* qs = sm;                               // [VT][LD]
  float* ps = qs + VT * LD;                     // [VT][LDP]: the weights
  float* tops = ps + VT * LDP;                  // [4 warps][VT]: the rows' maxima over a warp's keys
  float* tiles = tops + 4 * VT;                 // [STAGES]: keys [KB][LD], values [KB][LDV]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, group = c.nh / c.nkv;
  const int blocks = (it.end - it.begin + KB - 1) / KB;
  auto fetch = [&](int b) {
    float* tile = tiles + (b % STAGES) * TILE;
    if (b < blocks) load_block<T>(tile, tile + KB * LD, kc, vc, c, it, it.begin + b * KB, hd, wide);
    cp_async_commit();
  };
  // (what leads to the queries is asked for before the first block's page is waited for)
  const int row = lane < it.vectors && lane < 16 * MT ? c.rows[it.i0 + (it.vector0 + lane) / group] : -1;
  if (STAGES > 1) fetch(0);
  const int first_unseen = load_queries<T>(q, c, it, hd, 16 * MT, row, qs, tiles);
  // of the rows 16 i + g and 16 i + g + 8: keys that are not the vector's begin at `limit`; maximum and this thread's share of the sum
  int limit[2 * MT];
  float m[2 * MT], l[2 * MT];
#pragma unroll
  for (int x = 0; x < 2 * MT; ++x) {
    limit[x] = __shfl_sync(0xffffffffu, first_unseen, 8 * x + g);
    m[x] = -INFINITY;
    l[x] = 0.0f;
  }
  float acc[MT][NT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[i][n][0] = acc[i][n][1] = acc[i][n][2] = acc[i][n][3] = 0.0f;
  for (int b = 0; b < blocks; ++b) {
    fetch(b + STAGES - 1);
    cp_async_wait<STAGES - 1>();
    __syncthreads();
    const float* kt = tiles + (b % STAGES) * TILE + warp * 8 * LD;
    const float* vt = tiles + (b % STAGES) * TILE + KB * LD;
    float s[MT][4], small[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = small[i][e] = 0.0f;
#pragma unroll 1
    for (int k0 = 0; k0 < D; k0 += 32) {
      float large[MT][4];
#pragma unroll
      for (int i = 0; i < MT; ++i) large[i][0] = large[i][1] = large[i][2] = large[i][3] = 0.0f;
#pragma unroll
      for (int k = k0; k < k0 + 32; k += 8) {
        if (D % 32 != 0 && k >= D) break;
        const float b0 = kt[g * LD + k + t], b1 = kt[g * LD + k + t + 4];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          uint32_t h[4], lo[4];
          load_a(qs + 16 * i * LD + k, LD, h, lo);
          product<EXACT>(large[i], small[i], h, lo, b0, b1);
        }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] += large[i][e];
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] += small[i][e];
    const int key = it.begin + b * KB + warp * 8 + 2 * t;
#pragma unroll
    for (int x = 0; x < 2 * MT; ++x) {
      float* two = s[x >> 1] + 2 * (x & 1);
      if (key >= limit[x]) two[0] = -INFINITY;
      if (key + 1 >= limit[x]) two[1] = -INFINITY;
      float top = fmaxf(two[0], two[1]);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (t == 0) tops[warp * VT + 8 * x + g] = top;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 2 * MT; ++x) {
      const int r = 8 * x + g;
      const float m_new = fmaxf(m[x], fmaxf(fmaxf(tops[r], tops[VT + r]), fmaxf(tops[2 * VT + r], tops[3 * VT + r])));
      const float base = m_new == -INFINITY ? 0.0f : m_new, f = prefix_exp2(m[x] - base);      // (0 on the first visible block)
      const float* two = s[x >> 1] + 2 * (x & 1);
      const float p0 = prefix_exp2(two[0] - base), p1 = prefix_exp2(two[1] - base);
      *reinterpret_cast<float2*>(ps + r * LDP + warp * 8 + 2 * t) = make_float2(p0, p1);
      l[x] = l[x] * f + (p0 + p1);
      m[x] = m_new;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[x >> 1][n][2 * (x & 1)] *= f;
        acc[x >> 1][n][2 * (x & 1) + 1] *= f;
      }
    }
    __syncthreads();
    uint32_t h[KB / 8][MT][4], lo[KB / 8][MT][4];
#pragma unroll
    for (int k = 0; k < KB / 8; ++k)
#pragma unroll
      for (int i = 0; i < MT; ++i) load_a(ps + 16 * i * LDP + 8 * k, LDP, h[k][i], lo[k][i]);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (D % 32 != 0 && warp + 4 * n >= D / 8) break;
      const int dim = (warp + 4 * n) * 8 + g;
      float large[MT][4], rest[MT][4];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) large[i][e] = rest[i][e] = 0.0f;
#pragma unroll
      for (int k = 0; k < KB / 8; ++k) {
        const float b0 = vt[(8 * k + t) * LDV + dim], b1 = vt[(8 * k + t + 4) * LDV + dim];
#pragma unroll
        for (int i = 0; i < MT; ++i) product<EXACT>(large[i], rest[i], h[k][i], lo[k][i], b0, b1);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][n][e] += large[i][e] + rest[i][e];
    }
    __syncthreads();
  }
  // the rows' sums over the lanes and the warps (their maxima are the same everywhere)
#pragma unroll
  for (int x = 0; x < 2 * MT; ++x) {
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    if (t == 0) tops[warp * VT + 8 * x + g] = l[x];
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < 2 * MT; ++x) {
    const int r = 8 * x + g;
    if (r >= it.vectors) continue;
    const long long place = place_of(c, it, r);
    if (warp == 0 && t == 0) c.part_ml[place] = part_of(m[x], (tops[r] + tops[VT + r]) + (tops[2 * VT + r] + tops[3 * VT + r]));
    if (blocks > 0)
#pragma unroll
      for (int n = 0; n < NT; ++n)
        if (D % 32 == 0 || warp + 4 * n < D / 8)
          *reinterpret_cast<float2*>(c.part_acc + place * D + (warp + 4 * n) * 8 + 2 * t) = make_float2(acc[x >> 1][n][2 * (x & 1)], acc[x >> 1][n][2 * (x & 1) + 1]);
  }
  __syncthreads();                              // (a CTA may have another tile)
}
template <typename T>
__device__ __forceinline__ void attend(const T* __restrict__ q, const T* __restrict__ kc, const T* __restrict__ vc, const PrefixCall& c,
                                       const PrefixItem& it, int hd, bool wide, float* sm) {
  if (it.vectors <= 16) attend<T, 1>(q, kc, vc, c, it, hd, wide, sm);
  else attend<T, 2>(q, kc, vc, c, it, hd, wide, sm);
}

// grid: the shared keys' CTAs (split, KV head, tile, group), then the rows' own (split, KV head and part of its query heads, row).
template <typename T>
__global__ void __launch_bounds__(THREADS)
prefix_any_kernel(const T* __restrict__ q, const T* __restrict__ kc, const T* __restrict__ vc, const PrefixCall c, int hd, bool wide) {
  extern __shared__ __align__(16) float sm[];
  if (threadIdx.x < 32) prefetch_indices(c);
  pdl_wait();
  pdl_launch_dependents();
  const int group = c.nh / c.nkv;
  const int shared_ctas = c.splits_shared * c.nkv * c.tiles * c.n_groups;
  int b = blockIdx.x;
  PrefixItem it;
  int split, splits;
  if (b < shared_ctas) {
    splits = c.splits_shared;
    split = b % splits;
    b /= splits;
    it.kvh = b % c.nkv;
    b /= c.nkv;
    const int g = b / c.tiles;
    const int2 rows = rows_of_group(c, g);
    if (rows.y == 0) return;
    const int keys = shared_of_group(c, g);
    it.table = c.block_table + static_cast<long long>(c.rows[rows.x]) * c.table_stride;
    it.i0 = rows.x;
    it.slot = split;
    const int per = ((keys + KB - 1) / KB + splits - 1) / splits * KB;
    it.begin = min(keys, split * per);
    it.end = min(keys, it.begin + per);
    for (int tile = b % c.tiles; tile * VT < rows.y * group; tile += c.tiles) {
      it.vector0 = tile * VT;
      it.vectors = min(VT, rows.y * group - tile * VT);
      attend<T>(q, kc, vc, c, it, hd, wide, sm);
    }
    return;
  }
  b -= shared_ctas;
  splits = c.splits_own;
  split = b % splits;
  b /= splits;
  const int parts = (group + VT - 1) / VT;
  it.vector0 = b % parts * VT;
  b /= parts;
  it.kvh = b % c.nkv;
  it.i0 = b / c.nkv;
  it.vectors = min(VT, group - it.vector0);
  const int g = group_of_row(c, it.i0), row = c.rows[it.i0];
  const int keys = keys_of_row(c, row);
  const int from = min(keys, g < 0 ? 0 : shared_of_group(c, g));
  if (g < 0) {                                  // (a row in front of the first group: nobody else writes its other slots)
    for (int i = threadIdx.x; i < it.vectors * c.splits_shared; i += THREADS)
      c.part_ml[(static_cast<long long>(it.i0) * c.nh + it.kvh * group + it.vector0 + i / c.splits_shared) * prefix_splits(c) + i % c.splits_shared] =
          make_float2(-INFINITY, 0.0f);
  }
  it.table = c.block_table + static_cast<long long>(row) * c.table_stride;
  it.slot = c.splits_shared + split;
  const int per = ((keys - from + KB - 1) / KB + splits - 1) / splits * KB;
  it.begin = min(keys, from + split * per);
  it.end = min(keys, it.begin + per);
  attend<T>(q, kc, vc, c, it, hd, wide, sm);
}

// Head `head` of the i-th row's query, whose token's place is `at`, against all of its keys by a CTA: a warp every WARPS-th key as it lies in the
// cache, dims on its lanes, softmax as the keys come.  (Not inlined, and its arguments copies: the call is rare.)
template <typename T, int WARPS>
__device__ __noinline__ void attend_again(const T* q, const T* __restrict__ kc, const T* __restrict__ vc, T* out, const PrefixCall c, int i, int head,
                                          int hd, JoinShared<D, WARPS>* left) {
  constexpr int PER = (D + 31) / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kvh = head / (c.nh / c.nkv);
  const int row = c.rows[i], keys = keys_of_row(c, row), g = group_of_row(c, i);
  const int shared = g < 0 ? 0 : min(keys, shared_of_group(c, g));
  const int* table = c.block_table + static_cast<long long>(row) * c.table_stride;
  const int* shared_table = g < 0 ? table : c.block_table + static_cast<long long>(c.rows[rows_of_group(c, g).x]) * c.table_stride;
  const long long at = (static_cast<long long>(c.cu_q[row]) * c.nh + head) * hd;
  float x[PER], o[PER], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    x[n] = lane + 32 * n < hd ? to_f32<T>(q[at + lane + 32 * n]) * c.scale_log2 : 0.0f;
    o[n] = 0.0f;
  }
  for (int key = warp; key < keys; key += WARPS) {
    const int page = (key < shared ? shared_table : table)[key / c.page_size];
    if (page < 0 || page >= c.pages) continue;                 // (the error word has been set)
    const long long line = ((static_cast<long long>(page) * c.nkv + kvh) * c.page_size + key % c.page_size) * hd;
    float s = 0.0f, v[PER];
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const bool there = lane + 32 * n < hd;
      v[n] = there ? to_f32<T>(vc[line + lane + 32 * n]) : 0.0f;
      if (there) s = fmaf(x[n], to_f32<T>(kc[line + lane + 32 * n]), s);
    }
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) s += __shfl_xor_sync(0xffffffffu, s, step);
    const float most = fmaxf(m, s), base = most == -INFINITY ? 0.0f : most;
    const float f = prefix_exp2(m - base), p = prefix_exp2(s - base);      // (f: 0 on the first key that is seen)
    l = fmaf(l, f, p);
    m = most;
#pragma unroll
    for (int n = 0; n < PER; ++n) o[n] = fmaf(p, v[n], o[n] * f);
  }
  __syncthreads();                              // (`left` has been read)
#pragma unroll
  for (int n = 0; n < PER; ++n)
    if (D % 32 == 0 || lane + 32 * n < D) left->row[warp][lane + 32 * n] = o[n];
  if (lane == 0) { left->row[warp][D] = m; left->row[warp][D + 1] = l; }
  __syncthreads();
  float most = -INFINITY, sum = 0.0f;
  for (int w = 0; w < WARPS; ++w) most = fmaxf(most, left->row[w][D]);
  const float base = most == -INFINITY ? 0.0f : most;
  for (int w = 0; w < WARPS; ++w) sum = fmaf(left->row[w][D + 1], prefix_exp2(left->row[w][D] - base), sum);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  for (int dim = threadIdx.x; dim < hd; dim += WARPS * 32) {
    float y = 0.0f;
    for (int w = 0; w < WARPS; ++w) y = fmaf(left->row[w][dim], prefix_exp2(left->row[w][D] - base), y);
    out[at + dim] = from_f32<T>(y * inv);
  }
}

// A vector's splits joined: grid (n_rows * nh).  (`out` may be `q`: a CTA reads and writes its own vector's place.)
template <typename T, int JOIN_WARPS>
__global__ void __launch_bounds__(JOIN_WARPS * 32)
prefix_any_join_kernel(const T* q, const T* __restrict__ kc, const T* __restrict__ vc, T* out, const PrefixCall c, int hd) {
  __shared__ __align__(16) JoinShared<D, JOIN_WARPS> left;
  const int i = static_cast<int>(blockIdx.x) / c.nh, head = static_cast<int>(blockIdx.x) - i * c.nh;
  T* dst = out + (static_cast<long long>(c.cu_q[c.rows[i]]) * c.nh + head) * hd;
  pdl_launch_dependents();
  pdl_wait();
  const int splits = prefix_splits(c);
  const long long vec = static_cast<long long>(blockIdx.x) * splits;
  const bool done = join_parts<D, JOIN_WARPS, true>(dst, hd, splits, [&](int p, const float2*& ml, const float*& acc) {
    ml = c.part_ml + vec + p;
    acc = c.part_acc + (vec + p) * D;
  }, left);
  if (!done) attend_again<T, JOIN_WARPS>(q, kc, vc, out, c, i, head, hd, &left);
}

template <typename T>
static int launch(const void* q, const void* kc, const void* vc, void* out, const PrefixCall& c, int hd, int sms, cudaStream_t stream) {
  static bool seen[16];
  int rc = prefix_smem_limit(prefix_any_kernel<T>, SMEM, seen);
  if (rc != 0) return rc;
  const int parts = (c.nh / c.nkv + VT - 1) / VT;
  const long long ctas = static_cast<long long>(c.splits_shared) * c.nkv * c.tiles * c.n_groups + static_cast<long long>(c.splits_own) * parts * c.nkv * c.n_rows;
  const long long vectors = static_cast<long long>(c.n_rows) * c.nh;
  if (ctas > INT32_MAX || vectors > INT32_MAX) return B200_BAD_SIZE;
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const bool wide = sizeof(T) == 4 && hd % 4 == 0 && aligned(kc) && aligned(vc);
  rc = b200_launch(prefix_any_kernel<T>, dim3(static_cast<unsigned>(ctas)), dim3(THREADS), SMEM, stream, 0, static_cast<const T*>(q), static_cast<const T*>(kc),
                   static_cast<const T*>(vc), c, hd, wide);
  if (rc != 0) return rc;
  // (16 warps' rows of 512 floats: 33 KB)
  const int warps = join_warps_of(vectors, sms);
  return b200_launch(warps == 16 ? prefix_any_join_kernel<T, 16> : warps == 8 ? prefix_any_join_kernel<T, 8> : warps == 4 ? prefix_any_join_kernel<T, 4> : prefix_any_join_kernel<T, 2>,
                     dim3(static_cast<unsigned>(vectors)), dim3(warps * 32), 0, stream, 0, static_cast<const T*>(q), static_cast<const T*>(kc),
                     static_cast<const T*>(vc), static_cast<T*>(out), c, hd);
}

B200_EXPORT int b200_prefix_attention_smem() { return SMEM; }

// `scratch`: (HEAD_DIM + 2) floats for each of n_rows * nh * (splits_shared + splits_own), on a 16-byte boundary.
B200_EXPORT int b200_prefix_attention(const void* q, const void* k_cache, const void* v_cache, void* out, float* scratch, const int* block_table,
                                      int table_stride, const int* cu_q, const int* kv_len, const int* rows, int n_rows, const int* groups,
                                      int n_groups, int nh, int nkv, int page_size, int pages, float scale, int splits_shared, int splits_own,
                                      int tiles, int dtype, int head_dim, int sms, int* err, cudaStream_t stream) {
  if (n_rows <= 0) return 0;
  if (nh <= 0 || nkv <= 0 || nh % nkv != 0 || page_size <= 0 || pages <= 0 || table_stride <= 0 || n_groups < 0) return B200_BAD_SIZE;
  if (splits_shared < 1 || splits_own < 1 || tiles < 1 || head_dim <= 0 || head_dim > D || (head_dim & 1) || sms < 1) return B200_BAD_SIZE;
  if (!prefix_can_be_served({q, k_cache, v_cache, out, scratch, block_table, cu_q, kv_len, rows, err}, groups, n_groups, table_stride, page_size))
    return B200_BAD_SIZE;
  const PrefixCall c = {block_table, cu_q, kv_len, rows, reinterpret_cast<const int2*>(groups), scratch,
                        reinterpret_cast<float2*>(scratch + static_cast<size_t>(n_rows) * nh * (splits_shared + splits_own) * D), err, table_stride, n_rows,
                        n_groups, nh, nkv, page_size, pages, splits_shared, splits_own, tiles, scale * 1.4426950408889634f};
  if (dtype == B200_F32) return launch<float>(q, k_cache, v_cache, out, c, head_dim, sms, stream);
  if (dtype == B200_BF16) return launch<__nv_bfloat16>(q, k_cache, v_cache, out, c, head_dim, sms, stream);
  return B200_BAD_DTYPE;
}
