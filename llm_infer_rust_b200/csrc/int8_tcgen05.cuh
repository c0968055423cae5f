// Products in 8-bit integers on the fifth-generation tensor cores: tiles of tokens x columns, 32-bit integer sums in tensor
// memory, scales and gate as the epilogue.
//
// A tile is 128 tokens a CTA x BN columns (INT8_GLU: BN / 2 gate columns and the same BN / 2 up columns), k in blocks of 128
// bytes.  Warps:
//   warp 0      one lane feeds a ring of 6 stages with TMA (128-byte swizzle): a box of 128 tokens and two of 64 weight rows
//   warp 1      allocates tensor memory for two accumulators; one lane issues tcgen05.mma (kind::i8, K 32, four a stage)
//   warps 2-5   read their 32 lanes of tensor memory, multiply by the scales, round, turn the tile's rows through shared
//               memory and store whole 128-byte pieces of them
// Three ways to run it:
//   PAIRS    CG = 2, 256 tokens x 256 columns on two CTAs (each holds its 128 tokens and half of the weight rows, the
//            first one's MMAs read both): half the bytes per product that a CTA of its own would have to fetch, for the many
//            tiles of prompts.  Persistent: the epilogue of a tile runs under the MMAs of the next.
//   SINGLE   CG = 1, 128 x 128, persistent.
//   SPLIT    CG = 1, 128 x 128, a cluster of S CTAs shares a tile's k.  Each CTA sends its sums to the CTAs that own the
//            columns (distributed shared memory), which add them (integers: no order to keep) and finish.  For few tiles,
//            whose weights else come through few SMs.
// What lies beyond the matrices is zero-filled by TMA and masked at the store.  Every wait is bounded by the clock; one that
// runs out flags the engine's error word, and every path reaches the end, where tensor memory is given back.
#pragma once
#include <cuda.h>
#include <math.h>
#include <string.h>

#include "common.cuh"

enum : int { INT8_PLAIN = 0, INT8_GLU = 1 };

struct Int8ProductParams {
  const int8_t* q;           // [tokens, k], rows q_pitch bytes apart
  const float* s;            // [tokens]
  const int8_t* w;           // [rows, k], rows w_pitch bytes apart
  const float* c;            // [rows]
  const float* bias;         // [rows] or null
  void* out;                 // [tokens, n]
  int tokens, n, k;          // n: columns of out (INT8_GLU: w has 2 n rows)
  long long q_pitch, w_pitch;
  float limit, alpha;
  int* err;
};

namespace i8tc {

constexpr int BM = 128, BK = 128, STAGES = 6, THREADS = 192;
constexpr int A_BYTES = BM * BK, W_BYTES = 128 * BK, STAGE_BYTES = A_BYTES + W_BYTES;      // 32 KB
constexpr int GROUP_M = 16;                       // tiles of tokens that are walked over before the next columns

template <int CG> struct Shape {
  static constexpr int BN = CG == 2 ? 256 : 128;
  static constexpr int TURN = 4 * 32 * 128;                                     // a warp's 32 rows x 128 bytes
  static constexpr int SCALES = 4 * BN * 8;                                     // a warp's scales and bias
  static constexpr int SMEM = 1024 + STAGES * STAGE_BYTES + TURN + SCALES + (2 * STAGES + 4) * 8 + 16;
};
static_assert(Shape<2>::SMEM <= 227 * 1024, "shared memory of a CTA");

__device__ __forceinline__ void mbar_init(uint64_t* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t cta_address(const void* p, uint32_t rank) {     // the same place in another CTA of the cluster
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void mbar_arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_addr) : "memory");
}
template <int CG> __device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n"
                 ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n"
                 ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* map, int x, int y) {          // into the second-level cache
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];\n" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y) : "memory");
}
// K-major tile, 128-byte swizzle: rows of 128 bytes, groups of 8 rows 1,024 bytes apart; `addr` + 32 for every 32 k.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
  const uint32_t lo = ((addr >> 4) & 0x3FFFu) | (1u << 16);
  const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}
// 32-bit integer sums, signed 8-bit A and B, both K-major.
template <int CG> __host__ __device__ constexpr uint32_t instr_desc() {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((Shape<CG>::BN >> 3) << 17) | ((CG * BM >> 4) << 24);
}
template <int CG> __device__ __forceinline__ void mma_i8(uint32_t tmem_c, uint64_t a, uint64_t b, uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(tmem_c), "l"(a), "l"(b), "r"(instr_desc<CG>()), "r"(accumulate) : "memory");
  else
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(tmem_c), "l"(a), "l"(b), "r"(instr_desc<CG>()), "r"(accumulate) : "memory");
}
// The barrier (of both CTAs of a pair) is arrived on when all earlier MMAs are done.
template <int CG> __device__ __forceinline__ void mma_commit(uint64_t* bar) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n"
                 ::"r"(smem_u32(bar)), "h"(static_cast<uint16_t>(3)) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, int (&r)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
               "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                 "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                 "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
// mbar_wait for arrivals out of the other CTA of a pair.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity, int* err) {
  uint64_t start = 0;
  for (uint32_t polls = 1;; ++polls) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    if (ok) return true;
    if ((polls & 63u) == 0u) {
      const uint64_t now = global_ns();
      if (start == 0) start = now;
      if (now - start > 1000000000ull) {
        atomicOr(err, B200_ERR_WAIT_TIMEOUT);
        return false;
      }
    }
  }
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}

// Where a tile is: columns in order, GROUP_M tiles of tokens a column, so that CTAs that run together share weights and tokens.
__device__ __forceinline__ void tile_at(int tile, int m_tiles, int n_tiles, int& m, int& n) {
  const int first = tile / (GROUP_M * n_tiles) * GROUP_M, in = tile % (GROUP_M * n_tiles);
  const int rows = min(GROUP_M, m_tiles - first);
  m = first + in % rows;
  n = in / rows;
}

template <typename T> __device__ __forceinline__ uint32_t pack_word(const float* y);
template <> __device__ __forceinline__ uint32_t pack_word<float>(const float* y) { return __float_as_uint(y[0]); }
template <> __device__ __forceinline__ uint32_t pack_word<__nv_bfloat16>(const float* y) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(y[0], y[1]);
  return *reinterpret_cast<const uint32_t*>(&p);
}

template <typename T, int MODE, int CG, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1)
product_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap wmap, const Int8ProductParams P) {
  constexpr int BN = Shape<CG>::BN;
  constexpr int OUT = MODE == INT8_GLU ? BN / 2 : BN;                           // columns of the result a tile
  extern __shared__ unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* turn = ring + STAGES * STAGE_BYTES;
  float* scales = reinterpret_cast<float*>(turn + Shape<CG>::TURN);
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<unsigned char*>(scales) + Shape<CG>::SCALES);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;          // [2]
  uint64_t* acc_empty = acc_full + 2;           // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 || SPLIT ? cluster_rank() : 0u;
  uint32_t ranks = 1;
  if (SPLIT) asm volatile("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(ranks));
  const int m_tiles = (P.tokens + CG * BM - 1) / (CG * BM), n_tiles = (P.n + OUT - 1) / OUT, tiles = m_tiles * n_tiles;
  const int all_kb = (P.k + BK - 1) / BK;
  const int kb0 = SPLIT ? static_cast<int>(rank) * all_kb / static_cast<int>(ranks) : 0;
  const int kb1 = SPLIT ? (static_cast<int>(rank) + 1) * all_kb / static_cast<int>(ranks) : all_kb;
  const int first = SPLIT ? blockIdx.x / ranks : blockIdx.x / CG, step = SPLIT ? gridDim.x / ranks : gridDim.x / CG;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(acc_full + a, 1); mbar_init(acc_empty + a, 4 * CG); }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 1) {                                                              // the whole warp allocates tensor memory
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)), "r"(2 * BN) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)), "r"(2 * BN) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();                                                  // the pair's barriers exist
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();

  // the weight rows of a tile that this CTA fetches (two boxes of 64)
  auto weight_row = [&](int n, int box) {
    if (MODE == INT8_GLU) return CG == 2 ? (rank ? P.n : 0) + n * OUT + box * 64 : (box ? P.n : 0) + n * OUT;
    return n * OUT + static_cast<int>(CG == 2 ? rank : 0) * 128 + box * 64;
  };

  if (warp == 0) {
    if (lane == 0) {
      // The first weights start for the second-level cache before the dependency wait; nothing is read before it.
      int m, n;
      if (first < tiles) {
        tile_at(first, m_tiles, n_tiles, m, n);
        for (int kb = kb0; kb < kb1 && kb < kb0 + STAGES; ++kb)
          for (int box = 0; box < 2; ++box) tma_prefetch(&wmap, kb * BK, weight_row(n, box));
      }
      pdl_wait();
      int it = 0;                                                               // k-blocks fetched so far, over all tiles
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += step) {
        tile_at(tile, m_tiles, n_tiles, m, n);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % STAGES, use = it / STAGES;
          if (use > 0 && !mbar_wait(empty + s, (use - 1) & 1, P.err)) { ok = false; break; }
          unsigned char* st = ring + s * STAGE_BYTES;
          const uint32_t bar = CG == 2 ? cta_address(full + s, 0) : smem_u32(full + s);
          if (rank == 0 || CG == 1) mbar_expect_tx(full + s, CG * STAGE_BYTES);
          tma_load<CG>(st, &qmap, kb * BK, (m * CG + static_cast<int>(CG == 2 ? rank : 0)) * BM, bar);
          tma_load<CG>(st + A_BYTES, &wmap, kb * BK, weight_row(n, 0), bar);
          tma_load<CG>(st + A_BYTES + W_BYTES / 2, &wmap, kb * BK, weight_row(n, 1), bar);
        }
      }
    }
  } else if (warp == 1) {
    pdl_wait();
    if (lane == 0 && (CG == 1 || rank == 0)) {
      int it = 0, local = 0;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += step, ++local) {
        const int acc = local & 1, use = local >> 1;
        // (the epilogues have read this accumulator)
        if (use > 0) ok = CG == 2 ? mbar_wait_cluster(acc_empty + acc, (use - 1) & 1, P.err) : mbar_wait(acc_empty + acc, (use - 1) & 1, P.err);
        if (!ok) break;
        tc_fence_after();
        const uint32_t tmem_c = tmem_base + acc * BN;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % STAGES;
          ok = mbar_wait(full + s, (it / STAGES) & 1, P.err);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a = smem_u32(ring + s * STAGE_BYTES), b = a + A_BYTES;
#pragma unroll
          for (int k = 0; k < BK / 32; ++k) mma_i8<CG>(tmem_c, smem_desc(a + k * 32), smem_desc(b + k * 32), (kb > kb0 || k > 0) ? 1u : 0u);
          mma_commit<CG>(empty + s);                                            // the stage is free when these MMAs have read it
        }
        mma_commit<CG>(acc_full + acc);                                         // the tile's sums are complete
      }
    }
  } else if (!SPLIT) {
    pdl_wait();
    const int quarter = warp & 3;
    unsigned char* mine = turn + quarter * (32 * 128);
    float* sc = scales + quarter * (2 * BN);                                    // scales, then bias, in the accumulator's order
    int local = 0;
    T* out = static_cast<T*>(P.out);
    const bool whole = (reinterpret_cast<uintptr_t>(out) | (static_cast<size_t>(P.n) * sizeof(T))) % 16 == 0;
    constexpr int PIECE = 128 / sizeof(T);                                      // columns that are turned at once
    for (int tile = first; tile < tiles; tile += step, ++local) {
      int m, n;
      tile_at(tile, m_tiles, n_tiles, m, n);
      const int acc = local & 1;
      const int row0 = (m * CG + static_cast<int>(CG == 2 ? rank : 0)) * BM + quarter * 32;
      const int rows = min(32, P.tokens - row0);
      __syncwarp();
      for (int i = lane; i < BN; i += 32) {
        const int half = MODE == INT8_GLU ? i / OUT : 0, col = n * OUT + (MODE == INT8_GLU ? i % OUT : i);
        sc[i] = col < P.n ? P.c[half * P.n + col] : 0.0f;
        sc[BN + i] = P.bias && col < P.n ? P.bias[half * P.n + col] : 0.0f;
      }
      const float s = lane < rows ? P.s[row0 + lane] : 0.0f;
      __syncwarp();
      if (!mbar_wait(acc_full + acc, (local >> 1) & 1, P.err)) break;
      tc_fence_after();
      const uint32_t base = tmem_base + acc * BN + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
      for (int p = 0; p < OUT / PIECE; ++p) {
        const int col0 = n * OUT + p * PIECE;
        if (rows <= 0 || col0 >= P.n) break;                                    // (the whole warp)
#pragma unroll
        for (int h = 0; h < PIECE / 32; ++h) {
          const int at = p * PIECE + h * 32;
          int g[32], u[MODE == INT8_GLU ? 32 : 1];
          tmem_ld32(base + at, g);
          if constexpr (MODE == INT8_GLU) tmem_ld32(base + OUT + at, u);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; e += 16 / sizeof(T)) {
            uint4 piece;
            uint32_t* words = reinterpret_cast<uint32_t*>(&piece);
            constexpr int A_WORD = 4 / sizeof(T);
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              float y[A_WORD];
#pragma unroll
              for (int z = 0; z < A_WORD; ++z) {
                const int j = e + v * A_WORD + z;
                y[z] = fmaf(static_cast<float>(g[j]), s * sc[at + j], sc[BN + at + j]);
                if constexpr (MODE == INT8_GLU)
                  y[z] = glu_product(y[z], fmaf(static_cast<float>(u[j]), s * sc[OUT + at + j], sc[BN + OUT + at + j]), P.limit, P.alpha);
              }
              words[v] = pack_word<T>(y);
            }
            const int chunk = (h * 32 + e) * static_cast<int>(sizeof(T)) / 16;
            *reinterpret_cast<uint4*>(mine + lane * 128 + ((chunk ^ (lane & 7)) * 16)) = piece;
          }
        }
        __syncwarp();
        if (whole && col0 + PIECE <= P.n) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + lane / 8, chunk = lane % 8;
            if (r < rows)
              *reinterpret_cast<uint4*>(out + static_cast<size_t>(row0 + r) * P.n + col0 + chunk * (16 / sizeof(T))) =
                  *reinterpret_cast<const uint4*>(mine + r * 128 + ((chunk ^ (r & 7)) * 16));
          }
        } else {
          const int cols = min(PIECE, P.n - col0);
          for (int r = 0; r < rows; ++r)
            for (int c = lane; c < cols; c += 32) {
              const int byte = c * static_cast<int>(sizeof(T));
              out[static_cast<size_t>(row0 + r) * P.n + col0 + c] =
                  *reinterpret_cast<const T*>(mine + r * 128 + (((byte / 16) ^ (r & 7)) * 16) + byte % 16);
            }
        }
        __syncwarp();
      }
      tc_fence_before();                                                        // the loads of this accumulator are done
      __syncwarp();
      if (lane == 0) mbar_arrive_at(CG == 2 ? cta_address(acc_empty + acc, 0) : cta_address(acc_empty + acc, cluster_rank()));
    }
  } else {
    pdl_wait();
    if (first < tiles) mbar_wait(acc_full, 0, P.err);                           // (one tile a cluster)
    tc_fence_after();
  }

  if constexpr (SPLIT) {
    // Everybody's MMAs have read their rings, which take the others' sums now: [from][columns / 4][128 rows][4].
    __syncwarp();
    cluster_sync();
    int* sums = reinterpret_cast<int*>(ring);
    const int width = BN / static_cast<int>(ranks);                             // columns that a CTA owns (of gate and up each half)
    const int half = MODE == INT8_GLU ? OUT : BN, own = MODE == INT8_GLU ? width / 2 : width;
    int m, n;
    tile_at(first, m_tiles, n_tiles, m, n);
    const int rows = min(BM, P.tokens - m * BM);
    constexpr int QUAD = BM * 4;                                                // ints of four columns
    if (warp >= 2) {
      const int quarter = warp & 3, row = quarter * 32 + lane;
      if (quarter * 32 < rows) {
        const uint32_t base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
        for (int c = 0; c < BN; c += 32) {
          int v[32];
          tmem_ld32(base + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const int col = c + e, in = MODE == INT8_GLU ? col % half : col;
            const int to = in / own, quad = ((MODE == INT8_GLU && col >= half ? own : 0) + in % own) / 4;
            const uint32_t dst = cta_address(sums + (rank * (width / 4) + quad) * QUAD + row * 4, to);
            if (row < rows)
              asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(dst), "r"(v[e]), "r"(v[e + 1]), "r"(v[e + 2]), "r"(v[e + 3]) : "memory");
          }
        }
      }
    }
    __syncwarp();
    cluster_sync();
    pdl_wait();                                                                 // (every thread reads scales from here on)
    T* out = static_cast<T*>(P.out);
    const int quads = own / 4;
    for (int i = threadIdx.x; i < rows * quads; i += THREADS) {
      const int row = i / quads, quad = i % quads;
      const int col = n * OUT + static_cast<int>(rank) * own + quad * 4;
      if (col >= P.n) continue;
      const float s = P.s[m * BM + row];
      float y[2][4];
#pragma unroll
      for (int h = 0; h < (MODE == INT8_GLU ? 2 : 1); ++h) {
        int4 t = make_int4(0, 0, 0, 0);
        for (uint32_t from = 0; from < ranks; ++from) {
          const int4 v = *reinterpret_cast<const int4*>(sums + (from * (width / 4) + h * quads + quad) * QUAD + row * 4);
          t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w;
        }
        const int a[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = h * P.n + min(col + e, P.n - 1);
          y[h][e] = fmaf(static_cast<float>(a[e]), s * P.c[at], P.bias ? P.bias[at] : 0.0f);
        }
      }
      T* dst = out + static_cast<size_t>(m * BM + row) * P.n + col;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < P.n) dst[e] = from_f32<T>(MODE == INT8_GLU ? glu_product(y[0][e], y[1][e], P.limit, P.alpha) : y[0][e]);
    }
  }
  // Everybody meets here on every path; then the allocating warp gives the tensor memory back.
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  if (CG == 2) cluster_sync();                                                  // (the pair's MMAs and arrivals are over)
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(2 * BN) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(2 * BN) : "memory");
  }
}

// ------------------------------------------------------------------ host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The TMA descriptor of bytes [rows, k], rows `pitch` apart, fetched in boxes of box_rows x 128 bytes.
static int tensor_map(CUtensorMap* map, const void* matrix, long long rows, long long k, long long pitch, int box_rows) {
  static EncodeTiledFn encode = nullptr;
  if (encode == nullptr) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (fn == nullptr || found != cudaDriverEntryPointSuccess) return static_cast<int>(cudaErrorNotSupported);
    encode = reinterpret_cast<EncodeTiledFn>(fn);
  }
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(BK), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t elem_strides[2] = {1u, 1u};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(matrix), dims, strides, box, elem_strides,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 1000 + static_cast<int>(r);
}

template <typename T, int MODE, int CG, bool SPLIT>
static int launch(const Int8ProductParams& P, int blocks, int cluster, cudaStream_t stream) {
  static bool configured = false;
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(product_kernel<T, MODE, CG, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<CG>::SMEM);
    if (e != cudaSuccess) return static_cast<int>(e);
    configured = true;
  }
  CUtensorMap qmap, wmap;
  int rc = tensor_map(&qmap, P.q, P.tokens, P.k, P.q_pitch, BM);
  if (rc == 0) rc = tensor_map(&wmap, P.w, static_cast<long long>(P.n) * (MODE == INT8_GLU ? 2 : 1), P.k, P.w_pitch, 64);
  if (rc != 0) return rc;
  return b200_launch(product_kernel<T, MODE, CG, SPLIT>, dim3(blocks), dim3(THREADS), Shape<CG>::SMEM, stream, cluster, qmap, wmap, P);
}

// Which way a product goes (0 PAIRS, 1 SINGLE, S > 1 a cluster of S CTAs a tile).
static inline int route(int tokens, int n, int k, int mode, int sms) {
  const long long m1 = (tokens + 127) / 128, out1 = mode == INT8_GLU ? 64 : 128;
  const long long tiles = m1 * ((n + out1 - 1) / out1), pairs = (tokens + 255ll) / 256 * ((n + 2 * out1 - 1) / (2 * out1));
  if (tokens > 128 && pairs * 2 >= sms) return 0;
  const int kb = (k + BK - 1) / BK;
  int split = 1;
  while (split < 8 && tiles * split * 2 <= sms && split * 2 <= kb) split *= 2;
  return split;
}

template <typename T, int MODE> static int product(const Int8ProductParams& P, int sms, cudaStream_t stream) {
  const int way = route(P.tokens, P.n, P.k, MODE, sms);
  const int tall = way == 0 ? 256 : 128, wide = (way == 0 ? 256 : 128) / (MODE == INT8_GLU ? 2 : 1);
  const long long tiles = static_cast<long long>((P.tokens + tall - 1) / tall) * ((P.n + wide - 1) / wide);
  if (tiles > 0x3fffffff) return B200_BAD_SIZE;
  if (way == 0) return launch<T, MODE, 2, false>(P, 2 * static_cast<int>(tiles < sms / 2 ? tiles : sms / 2), 2, stream);
  if (way == 1) return launch<T, MODE, 1, false>(P, static_cast<int>(tiles < sms ? tiles : sms), 0, stream);
  return launch<T, MODE, 1, true>(P, static_cast<int>(tiles) * way, way, stream);
}

}  // namespace i8tc
