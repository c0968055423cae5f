// Decode attention behind shared prefixes (prefix.cuh) on CUDA cores: float32, and what the tensor-core kernels do not take
// (head sizes that are no multiple of 16, pages of no power of two, more than 16 query heads a KV head).  Compile with
// -DHEAD_DIM=<multiple of 16, at most 512>; the real head size may be smaller.
//
// A CTA has a tile of 32 query vectors and walks its split of the keys in blocks of 32, two blocks of keys and values on their
// way where they fit.  S = Q K^T: a thread owns 2 vectors x 4 keys, so that a row's maximum and sum stay in eight lanes of a
// warp; the weights go through shared memory, transposed; O += P V: a thread owns 4 vectors x every 16th group of four dims.
// Bound by the multiply-adds of the 32 vectors (a key of 128 dims in float32: 64 cycles of an SM, its bytes from memory 45).
#include "prefix.cuh"

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<head size, a multiple of 16>"
#endif
static_assert(HEAD_DIM % 16 == 0 && HEAD_DIM >= 16 && HEAD_DIM <= 512, "head sizes 16 to 512 in steps of 16");

constexpr int D = HEAD_DIM;
constexpr int VT = 32, KB = 32, THREADS = 128;
constexpr int LD = D + 4;                       // a padded row: eight rows' float4 lie in eight different groups of banks
constexpr int COLS = D / 4, PER = (COLS + 15) / 16;
constexpr int TILE = KB * LD;                   // floats of a block's keys (or values)
constexpr int FIXED = VT * LD + KB * (VT + 4) + VT;
constexpr int STAGES = (FIXED + 4 * TILE) * 4 <= 220 * 1024 ? 2 : 1;
constexpr int SMEM = (FIXED + STAGES * 2 * TILE) * 4;
static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

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
  float* vd = v + j * LD;
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

// One tile of up to 32 vectors against the item's keys; the results go to the vectors' slots.
template <typename T>
__device__ void attend(const T* __restrict__ q, const T* __restrict__ kc, const T* __restrict__ vc, const PrefixCall& c,
                       const PrefixItem& it, int hd, bool wide, float* sm) {
  float* qs = sm;                               // [VT][LD]
  float* pt = qs + VT * LD;                     // [KB][VT + 4]: the weights, a key's 32 in a row
  float* fs = pt + KB * (VT + 4);               // [VT]: what the accumulators are scaled by
  float* tiles = fs + VT;                       // [STAGES][2][KB][LD]
  const int group = c.nh / c.nkv;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < VT * D; i += THREADS) {
    const int r = i / D, dim = i - r * D;
    float x = 0.0f;
    if (r < it.vectors && dim < hd) {
      const int vec = it.vector0 + r;
      const int tok = c.cu_q[c.rows[it.i0 + vec / group]];
      x = to_f32<T>(q[(static_cast<long long>(tok) * c.nh + it.kvh * group + vec % group) * hd + dim]) * c.scale_log2;
    }
    qs[r * LD + dim] = x;
  }
  if (hd < D)                                   // the padded columns are zeros for good
    for (int i = threadIdx.x; i < STAGES * 2 * KB * (D - hd); i += THREADS) tiles[i / (D - hd) * LD + hd + i % (D - hd)] = 0.0f;

  const int v0 = (warp * 4 + (lane >> 3)) * 2, k0 = lane & 7;      // this thread's vectors v0, v0 + 1 and keys k0 + 8 n
  int limit[2];                                 // keys from here on are not this vector's
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    limit[x] = 0;
    if (v0 + x < it.vectors) limit[x] = min(it.end, keys_of_row(c, c.rows[it.i0 + (it.vector0 + v0 + x) / group]));
  }
  const int ov = (threadIdx.x >> 4) * 4, dg = threadIdx.x & 15;    // and of the output vectors ov .. ov + 3, columns dg + 16 n
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  float acc[4][PER][4];
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int n = 0; n < PER; ++n) acc[x][n][0] = acc[x][n][1] = acc[x][n][2] = acc[x][n][3] = 0.0f;

  const int blocks = (it.end - it.begin + KB - 1) / KB;
  auto fetch = [&](int b) {
    if (b < blocks) load_block<T>(tiles + (b % STAGES) * 2 * TILE, tiles + (b % STAGES) * 2 * TILE + TILE, kc, vc, c, it, it.begin + b * KB, hd, wide);
    cp_async_commit();
  };
  if (STAGES > 1) fetch(0);
  for (int b = 0; b < blocks; ++b) {
    fetch(b + STAGES - 1);
    cp_async_wait<STAGES - 1>();
    __syncthreads();
    const float* kt = tiles + (b % STAGES) * 2 * TILE;
    const float* vt = kt + TILE;
    float s[2][4] = {};
#pragma unroll 4
    for (int col = 0; col < COLS; ++col) {
      const float4 a0 = *reinterpret_cast<const float4*>(qs + v0 * LD + col * 4);
      const float4 a1 = *reinterpret_cast<const float4*>(qs + (v0 + 1) * LD + col * 4);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float4 k4 = *reinterpret_cast<const float4*>(kt + (k0 + 8 * n) * LD + col * 4);
        s[0][n] = fmaf(a0.x, k4.x, fmaf(a0.y, k4.y, fmaf(a0.z, k4.z, fmaf(a0.w, k4.w, s[0][n]))));
        s[1][n] = fmaf(a1.x, k4.x, fmaf(a1.y, k4.y, fmaf(a1.z, k4.z, fmaf(a1.w, k4.w, s[1][n]))));
      }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        if (it.begin + b * KB + k0 + 8 * n >= limit[x]) s[x][n] = -INFINITY;
        mx = fmaxf(mx, s[x][n]);
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float m_new = fmaxf(m[x], mx);
      const float base = m_new == -INFINITY ? 0.0f : m_new, f = fast_exp2(m[x] - base);     // (0 on the first visible block)
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float p = fast_exp2(s[x][n] - base);
        sum += p;
        pt[(k0 + 8 * n) * (VT + 4) + v0 + x] = p;
      }
      l[x] = l[x] * f + sum;                    // (this thread's share of the row's sum)
      m[x] = m_new;
      if (k0 == 0) fs[v0 + x] = f;
    }
    __syncthreads();
    const float4 f4 = *reinterpret_cast<const float4*>(fs + ov);
    const float f[4] = {f4.x, f4.y, f4.z, f4.w};
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int n = 0; n < PER; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[x][n][e] *= f[x];
#pragma unroll 4
    for (int key = 0; key < KB; ++key) {
      const float4 p4 = *reinterpret_cast<const float4*>(pt + key * (VT + 4) + ov);
      const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
      for (int n = 0; n < PER; ++n) {
        const int col = dg + 16 * n;
        if (COLS % 16 == 0 || col < COLS) {
          const float4 w = *reinterpret_cast<const float4*>(vt + key * LD + col * 4);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            acc[x][n][0] = fmaf(p[x], w.x, acc[x][n][0]);
            acc[x][n][1] = fmaf(p[x], w.y, acc[x][n][1]);
            acc[x][n][2] = fmaf(p[x], w.z, acc[x][n][2]);
            acc[x][n][3] = fmaf(p[x], w.w, acc[x][n][3]);
          }
        }
      }
    }
    __syncthreads();
  }
  const int splits = prefix_splits(c);
  auto place = [&](int r) {                     // of vector r's results
    const int vec = it.vector0 + r;
    return (static_cast<long long>(it.i0 + vec / group) * c.nh + it.kvh * group + vec % group) * splits + it.slot;
  };
#pragma unroll
  for (int x = 0; x < 2; ++x) {
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) l[x] += __shfl_xor_sync(0xffffffffu, l[x], o);
    if (k0 == 0 && v0 + x < it.vectors) c.part_ml[place(v0 + x)] = make_float2(m[x], l[x]);
  }
  if (blocks > 0) {
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (ov + x < it.vectors) {
        float* dst = c.part_acc + place(ov + x) * D;
#pragma unroll
        for (int n = 0; n < PER; ++n)
          if (COLS % 16 == 0 || dg + 16 * n < COLS) *reinterpret_cast<float4*>(dst + (dg + 16 * n) * 4) = make_float4(acc[x][n][0], acc[x][n][1], acc[x][n][2], acc[x][n][3]);
      }
  }
  __syncthreads();                              // (a CTA may have another tile)
}

// grid: the shared keys' CTAs (split, KV head, tile, group), then the rows' own (split, KV head and part of its query heads, row).
template <typename T>
__global__ void __launch_bounds__(THREADS)
prefix_any_kernel(const T* __restrict__ q, const T* __restrict__ kc, const T* __restrict__ vc, const PrefixCall c, int hd, bool wide) {
  extern __shared__ __align__(16) float sm[];
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

template <typename T>
static int launch(const void* q, const void* kc, const void* vc, void* out, const PrefixCall& c, int hd, cudaStream_t stream) {
  static bool seen[16];
  int rc = prefix_smem_limit(prefix_any_kernel<T>, SMEM, seen);
  if (rc != 0) return rc;
  const int parts = (c.nh / c.nkv + VT - 1) / VT;
  const long long ctas = static_cast<long long>(c.splits_shared) * c.nkv * c.tiles * c.n_groups + static_cast<long long>(c.splits_own) * parts * c.nkv * c.n_rows;
  if (ctas > INT32_MAX || c.nh > 65535) return B200_BAD_SIZE;
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const bool wide = sizeof(T) == 4 && hd % 4 == 0 && aligned(kc) && aligned(vc);
  prefix_any_kernel<T><<<static_cast<unsigned>(ctas), THREADS, SMEM, stream>>>(static_cast<const T*>(q), static_cast<const T*>(kc), static_cast<const T*>(vc), c, hd, wide);
  rc = b200_check_launch();
  if (rc != 0) return rc;
  return prefix_merge<T, D>(out, c, hd, stream);
}

B200_EXPORT int b200_prefix_attention_smem() { return SMEM; }

// `scratch`: (HEAD_DIM + 2) floats for each of n_rows * nh * (splits_shared + splits_own), on a 16-byte boundary.
B200_EXPORT int b200_prefix_attention(const void* q, const void* k_cache, const void* v_cache, void* out, float* scratch, const int* block_table,
                                      int table_stride, const int* cu_q, const int* kv_len, const int* rows, int n_rows, const int* groups,
                                      int n_groups, int nh, int nkv, int page_size, int pages, float scale, int splits_shared, int splits_own,
                                      int tiles, int dtype, int head_dim, int* err, cudaStream_t stream) {
  if (n_rows <= 0) return 0;
  if (nh <= 0 || nkv <= 0 || nh % nkv != 0 || page_size <= 0 || pages <= 0 || table_stride <= 0 || n_groups < 0) return B200_BAD_SIZE;
  if (splits_shared < 1 || splits_own < 1 || tiles < 1 || head_dim <= 0 || head_dim > D || (head_dim & 1)) return B200_BAD_SIZE;
  const PrefixCall c = {block_table, cu_q, kv_len, rows, reinterpret_cast<const int2*>(groups), scratch,
                        reinterpret_cast<float2*>(scratch + static_cast<size_t>(n_rows) * nh * (splits_shared + splits_own) * D), err, table_stride, n_rows,
                        n_groups, nh, nkv, page_size, pages, splits_shared, splits_own, tiles, scale * 1.4426950408889634f};
  if (dtype == B200_F32) return launch<float>(q, k_cache, v_cache, out, c, head_dim, stream);
  if (dtype == B200_BF16) return launch<__nv_bfloat16>(q, k_cache, v_cache, out, c, head_dim, stream);
  return B200_BAD_DTYPE;
}
