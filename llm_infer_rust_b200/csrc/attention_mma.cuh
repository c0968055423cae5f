// What the mma.sync attention kernels over the paged bfloat16 cache (attention_mma.cu, prefix_mma.cu) have in common, for one head
// size: the forms of a build, the fetch of a block of 32 keys and values, and its products with 16 query vectors.
#pragma once
#include <cuda.h>
#include <math.h>
#include <string.h>

#include "common.cuh"

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<head size, a multiple of 16>"
#endif
// A second form serves attention over a latent (compile with -DV_SHARED=1 -DV_DIM=<columns>): a token has ONE key row
// of HEAD_DIM columns (up to 512) that every query head reads, and its value is a range of V_DIM columns of that same
// row (from column ScoreForm::v_col0 on), so a block's tile is fetched once and serves both products.  The output
// goes to columns out_col0 .. out_col0 + V_DIM of rows out_width wide: values wider than 256 columns take several
// launches, each with the scores computed again.
//
// Values of another width than keys take a build with -DV_DIM=<multiple of 16, at most 256> (a block's tile then holds
// key boxes and value boxes of different counts).
//
// A build with -DDIFF=1 hands on the difference of a head's two maps (differential attention): the query vectors of a KV
// head are pairs, rows 2j and 2j + 1 the two maps of one head, and what is stored for the pair is
//     o / sqrt(mean(o^2) + diff_eps) * diff_gain,   o = a_(2j) - diff_lambda a_(2j + 1),
// in float from the softmax on and rounded once; an output row is half as many heads wide.
#ifndef V_SHARED
#define V_SHARED 0
#endif
#ifndef V_DIM
#define V_DIM HEAD_DIM
#endif
#ifndef DIFF
#define DIFF 0
#endif
static_assert(HEAD_DIM % 16 == 0 && HEAD_DIM >= 16 && HEAD_DIM <= (V_SHARED ? 512 : 256),
              "the tensor-core kernels take head sizes 16..256 in steps of 16 (keys of a shared row: up to 512)");
static_assert(V_DIM % 16 == 0 && V_DIM >= 16 && V_DIM <= 256 && (!V_SHARED || (V_DIM <= HEAD_DIM && !DIFF)),
              "values are 16..256 columns wide (of a shared row: some of the keys' own columns)");

typedef __nv_bfloat16 bf16;
constexpr int D = HEAD_DIM;
constexpr int DV = V_DIM;          // columns of a value and of an output tile
constexpr bool kShared = V_SHARED != 0;
constexpr bool kDiff = DIFF != 0;
constexpr int LD = D + 8;          // padded row of the query tile (16 bytes of padding): conflict-free ldmatrix
constexpr int KB = 32;             // keys per block
constexpr int NB = (D + 63) / 64;  // 64-dim (128-byte) column boxes per row
constexpr int HALF_BYTES = KB * 128;              // one column box of a block: 32 rows x 128 bytes
constexpr int NBV = kShared ? 0 : (DV + 63) / 64;                 // column boxes of a value row with a tile of its own
constexpr int TILE_BYTES = (NB + NBV) * HALF_BYTES;               // keys then values of one block (one tile for both)
constexpr int VALUE_CHUNKS = (kShared ? NB : NBV) * 8;            // 16-byte chunks of a row that holds values
constexpr int V_OFFSET = kShared ? 0 : NB * HALF_BYTES;           // where a block's values begin in its tile
constexpr int QROWS = 16;          // rows of the A operand: query heads of one KV head

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], const void* p) {
  const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p));
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], const void* p) {
  const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p));
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float fast_exp2(float x) {      // 2^x in one special-function instruction (-inf gives 0)
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// How a raw score q.k becomes the exponent of 2 that the softmax takes: score * scale_log2, or, with a soft-cap,
// cap_log2 * tanh(score * tanh_in) (cap_log2 = cap * log2(e), tanh_in = scale / cap; cap_log2 <= 0: no cap).
// split_p: the weights enter P.V as two bfloat16 terms, the rounded weight and what the rounding left, so that
// the product carries the weights to about 16 bits instead of 8.
// chunk C > 0: a query at position p also sees only keys from p - p % C on (its own block of C positions, counted
// from the sequence's start).  sinks (one float per query head, or null): exp(sink) joins the softmax's denominator.
struct ScoreForm {
  float scale_log2, tanh_in, cap_log2;
  int split_p;
  int chunk;
  const float* sinks;
  int v_col0;                  // shared rows: first column of the values
  int out_width, out_col0;     // an output row's width and the first column that this launch writes
  float diff_lambda, diff_gain, diff_eps;      // DIFF
};
// The sum of a row's weights with the sink's term (the row's maximum m is in log2 units).
__device__ __forceinline__ float with_sink(const ScoreForm& sf, int head, float m, float l) {
  return (sf.sinks != nullptr && l > 0.0f) ? l + exp2f(sf.sinks[head] * 1.4426950408889634f - m) : l;
}
__device__ __forceinline__ float tanh_by_exp2(float x) {     // 1 - 2 / (e^(2x) + 1): absolute error about 1e-7
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(e) : "f"(x * 2.8853900817779268f));
  return 1.0f - __fdividef(2.0f, e + 1.0f);
}
__device__ __forceinline__ uint32_t pack_bf16_rest(float lo, float hi, uint32_t& rest) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  const __nv_bfloat162 r = __floats2bfloat162_rn(lo - __low2float(v), hi - __high2float(v));
  rest = *reinterpret_cast<const uint32_t*>(&r);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// ---- mbarrier and bulk-copy primitives (the copy engine writes shared memory and signals the barrier)
__device__ __forceinline__ void mbar_init(uint64_t* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n"
               ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y) : "memory");
}

// Byte offset of (row r, 16-byte chunk c of the row's D dims) inside a tile of NB column boxes, each
// [32 rows][128 bytes] in the 128-byte swizzle (chunk index XOR row mod 8; tiles are 1024-byte aligned).
__device__ __forceinline__ int swz(int r, int c) {
  return (c >> 3) * HALF_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// One warp fetches keys [first_key, first_key + 32) of one KV head into `tile` (keys, then values).
// The block is cut into sub-blocks of `box_rows` rows (a power of two that divides 32 and the page
// size, so a sub-block never leaves its page); lane j issues the boxes of sub-block j with the page
// id `page` that it looked up one block earlier.  Sub-blocks that start at or beyond kv_end are skipped.
__device__ __forceinline__ void fetch_block(unsigned char* tile, const CUtensorMap* kmap, const CUtensorMap* vmap,
                                            int page, int page_size, int nkv, int kvh, int box_rows, int first_key,
                                            int kv_end, uint64_t* bar, int lane) {
  const int n_sub = (min(KB, kv_end - first_key) + box_rows - 1) / box_rows;
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");   // earlier reads and writes of the tile come first
  if (lane == 0) mbar_expect_tx(bar, static_cast<uint32_t>(n_sub) * (NB + NBV) * box_rows * 128u);
  __syncwarp();
  if (lane < n_sub) {
    const int key0 = first_key + lane * box_rows;
    const int y = kShared ? page * page_size + key0 % page_size          // one row a token for every head
                          : (page * nkv + kvh) * page_size + key0 % page_size;
#pragma unroll
    for (int h = 0; h < NB; ++h) {
      tma_load_2d(tile + h * HALF_BYTES + lane * box_rows * 128, kmap, h * 64, y, bar);
      if (h < NBV) tma_load_2d(tile + (NB + h) * HALF_BYTES + lane * box_rows * 128, vmap, h * 64, y, bar);
    }
#pragma unroll
    for (int h = NB; h < NBV; ++h)
      tma_load_2d(tile + (NB + h) * HALF_BYTES + lane * box_rows * 128, vmap, h * 64, y, bar);
  }
}

// Page id of the sub-block that this lane fetches in the block that starts at first_key.  It is loaded one
// block ahead of its use, so that the table's latency is off the copies' critical path.
__device__ __forceinline__ int lane_page(const int* __restrict__ table, int page_size, int box_rows, int first_key,
                                         int kv_end, int lane) {
  const int key0 = first_key + lane * box_rows;
  return (lane * box_rows < KB && key0 < kv_end) ? table[key0 / page_size] : 0;
}

// State of one warp: 16 query rows x D outputs in mma accumulator layout.
struct WarpAcc {
  float o[DV / 8][4];
  float m[2], l[2];          // rows lane/4 and lane/4 + 8; l is this thread's part of the row sum
  __device__ __forceinline__ void init() {
#pragma unroll
    for (int i = 0; i < DV / 8; ++i) { o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f; }
    m[0] = m[1] = -INFINITY; l[0] = l[1] = 0.0f;
  }
};

// One block of 32 keys against the 16 query rows in `qs`.  `qpos0/1`: position of the query in rows
// lane/4 and lane/4 + 8 (-1: the row is unused).  `sf`: scale, soft-cap and the form of the weights (ScoreForm).
// MASKED = false: the caller knows that every key of the block is visible to every used row of the warp.
// SHAPED: the score may be soft-capped and the weights split in two terms (`sf`); false: the plain form, which
// carries none of that code.
template <bool MASKED, bool SHAPED>
__device__ __forceinline__ void block_mma(const bf16* qs, const unsigned char* ks, const unsigned char* vs, int first_key, int kv_end,
                                          int window, int qpos0, int qpos1, const ScoreForm& sf, WarpAcc& st) {
  const int lane = threadIdx.x & 31;
  const int mi = lane >> 3, r8 = lane & 7;
  float s[4][4];
#pragma unroll
  for (int n = 0; n < 4; ++n) { s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f; }
#pragma unroll
  for (int ks16 = 0; ks16 < D / 16; ++ks16) {
    uint32_t a[4];
    ldmatrix_x4(a, qs + (lane & 15) * LD + ks16 * 16 + (lane >> 4) * 8);
#pragma unroll
    for (int n = 0; n < 4; n += 2) {
      uint32_t b[4];
      ldmatrix_x4(b, ks + swz(n * 8 + (mi >> 1) * 8 + r8, ks16 * 2 + (mi & 1)));
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
      bool v0 = qpos0 >= 0, v1 = qpos1 >= 0;
      if (MASKED) {
        const int key = first_key + n * 8 + t2 + e;
        const bool in_seq = key < kv_end;
        v0 = in_seq && v0 && key <= qpos0 && (window <= 0 || key > qpos0 - window) &&
             (sf.chunk <= 0 || key >= qpos0 - qpos0 % sf.chunk);
        v1 = in_seq && v1 && key <= qpos1 && (window <= 0 || key > qpos1 - window) &&
             (sf.chunk <= 0 || key >= qpos1 - qpos1 % sf.chunk);
      }
      float a0 = s[n][e] * sf.scale_log2, a1 = s[n][2 + e] * sf.scale_log2;
      if (SHAPED && sf.cap_log2 > 0.0f) {
        a0 = sf.cap_log2 * tanh_by_exp2(s[n][e] * sf.tanh_in);
        a1 = sf.cap_log2 * tanh_by_exp2(s[n][2 + e] * sf.tanh_in);
      }
      s[n][e] = v0 ? a0 : -INFINITY;
      s[n][2 + e] = v1 ? a1 : -INFINITY;
      mx0 = fmaxf(mx0, s[n][e]);
      mx1 = fmaxf(mx1, s[n][2 + e]);
    }
  }
  mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1)); mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
  mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1)); mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
  const float m0 = fmaxf(st.m[0], mx0), m1 = fmaxf(st.m[1], mx1);
  const float c0 = m0 == -INFINITY ? 1.0f : exp2f(st.m[0] - m0);      // exp2(-inf) = 0 on the first visible block
  const float c1 = m1 == -INFINITY ? 1.0f : exp2f(st.m[1] - m1);
  const float base0 = m0 == -INFINITY ? 0.0f : m0, base1 = m1 == -INFINITY ? 0.0f : m1;
  float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      s[n][e] = fast_exp2(s[n][e] - base0);          // a masked score is -inf: exp2 gives 0
      s[n][2 + e] = fast_exp2(s[n][2 + e] - base1);
      sum0 += s[n][e];
      sum1 += s[n][2 + e];
    }
  }
  st.m[0] = m0; st.m[1] = m1;
  st.l[0] = st.l[0] * c0 + sum0;
  st.l[1] = st.l[1] * c1 + sum1;
  if (__any_sync(0xffffffffu, c0 != 1.0f || c1 != 1.0f)) {       // no row's maximum moved: nothing to rescale
#pragma unroll
    for (int i = 0; i < DV / 8; ++i) { st.o[i][0] *= c0; st.o[i][1] *= c0; st.o[i][2] *= c1; st.o[i][3] *= c1; }
  }
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    uint32_t a[4], rest[4] = {0u, 0u, 0u, 0u};
    if constexpr (SHAPED) {
      a[0] = pack_bf16_rest(s[2 * kk][0], s[2 * kk][1], rest[0]);
      a[1] = pack_bf16_rest(s[2 * kk][2], s[2 * kk][3], rest[1]);
      a[2] = pack_bf16_rest(s[2 * kk + 1][0], s[2 * kk + 1][1], rest[2]);
      a[3] = pack_bf16_rest(s[2 * kk + 1][2], s[2 * kk + 1][3], rest[3]);
    } else {
      a[0] = pack_bf16(s[2 * kk][0], s[2 * kk][1]);
      a[1] = pack_bf16(s[2 * kk][2], s[2 * kk][3]);
      a[2] = pack_bf16(s[2 * kk + 1][0], s[2 * kk + 1][1]);
      a[3] = pack_bf16(s[2 * kk + 1][2], s[2 * kk + 1][3]);
    }
    const int v_chunk0 = kShared ? sf.v_col0 >> 3 : 0;
#pragma unroll
    for (int dn = 0; dn < DV / 8; dn += 2) {
      uint32_t b[4];
      ldmatrix_x4_trans(b, vs + swz(kk * 16 + (mi & 1) * 8 + r8, v_chunk0 + dn + (mi >> 1)));
      mma_bf16(st.o[dn], a, b[0], b[1]);
      mma_bf16(st.o[dn + 1], a, b[2], b[3]);
      if (SHAPED && sf.split_p) {
        mma_bf16(st.o[dn], rest, b[0], b[1]);
        mma_bf16(st.o[dn + 1], rest, b[2], b[3]);
      }
    }
  }
}
