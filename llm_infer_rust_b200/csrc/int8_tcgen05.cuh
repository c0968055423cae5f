// Products in 8-bit integers on the fifth-generation tensor cores: tiles of tokens x columns, 32-bit integer sums in tensor
// memory, scales and gate as the epilogue.
//
// A tile is 128 tokens a CTA x BN columns (INT8_GLU: BN / 2 gate columns and the same BN / 2 up columns), k in blocks of 128
// bytes.  Warps:
//   warp 0      one lane feeds a ring of stages with TMA (128-byte swizzle): a box of weight rows (or of gate and of up rows) for
//               each of a stage's blocks of k
//   warp 10     the same for the tokens
//   warp 1      allocates tensor memory for two accumulators; one lane issues tcgen05.mma (kind::i8, K 32, four a block)
//   warps 2-9   read their 32 lanes of tensor memory (two warps a quarter, every other 32 columns), multiply by the scales,
//               round, turn 32 x 32 results through shared memory and store pieces of rows
// Three ways to run it:
//   PAIRS    CG = 2, 256 tokens x up to 256 columns on two CTAs (each holds its 128 tokens and half of the weight rows, the
//            first one's MMAs read both): half the bytes per product that a CTA of its own would have to fetch, for the many
//            tiles of prompts.  Persistent: the epilogue of a tile runs under the MMAs of the next.
//   SINGLE   CG = 1, 128 x BN, persistent; BN is chosen so that the SMs get equal shares of the weights.
//   SPLIT    CG = 1, 128 x BN, a cluster of S CTAs shares a tile's k.  Each CTA sends its sums to the CTAs that own the
//            columns (distributed shared memory), which add them (integers: no order to keep) and finish.  For few tiles,
//            whose weights else come through few SMs.
// Token rows: a box is as high as there are tokens (to 8), and the last tile of 128 begins so that it ends with the tokens
// (rows it shares with the tile before are not stored again): TMA takes longer to fill rows outside a matrix with zeros
// than to fetch them.  Rows of the MMA's 128 beyond the box hold whatever lies there; sums of other rows do not see them.
// What lies beyond the matrices otherwise is zero-filled by TMA and masked at the store.  Every wait is bounded by the clock;
// one that runs out flags the engine's error word, and every path reaches the end, where tensor memory is given back.
#pragma once
#include <cuda.h>
#include <math.h>
#include <string.h>
#include <type_traits>

#include "int8_common.cuh"

namespace i8tc {

constexpr int BM = 128, BK = 128, MAX_STAGES = 16, EPI_WARPS = 8, PARTS = EPI_WARPS / 4, THREADS = (3 + EPI_WARPS) * 32;
constexpr int GROUP_M = 16;                       // tiles of tokens that are walked over before the next columns
constexpr int ACC = 256;                          // columns of tensor memory of an accumulator
constexpr int SCALES = 8192;                      // each warp's scales and bias: [pieces][gate, up][scale, bias][32]
template <typename T> constexpr int turn_bytes() { return EPI_WARPS * 32 * 32 * static_cast<int>(sizeof(T)); }        // a warp's 32 rows x 32 results
template <typename T> constexpr int smem_fixed() { return 1024 + turn_bytes<T>() + SCALES + (2 * MAX_STAGES + 4) * 8 + 16; }
constexpr int SMEM_MOST = 227 * 1024;

// How a product is cut up.
struct Plan {
  int way;                   // 0 PAIRS, 1 SINGLE, S > 1 a cluster of S CTAs a tile
  int bn;                    // columns of the accumulator (INT8_GLU: half of them gate columns)
  int box;                   // tokens that are fetched a tile
  int sub;                   // blocks of k a stage
  int stages, stage_bytes;
};

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
// An accumulator is handed back when its loads have completed (the caller has waited for them): relaxed, because a release over
// the cluster would first wait for the tile's stores.
template <int CG> __device__ __forceinline__ void mbar_hand_back(uint64_t* bar) {
  if constexpr (CG == 2) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(cta_address(bar, 0)) : "memory");
  else asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
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
template <int CG> __device__ __forceinline__ uint32_t instr_desc(int bn) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(bn >> 3) << 17) | ((CG * BM >> 4) << 24);
}
template <int CG> __device__ __forceinline__ void mma_i8(uint32_t tmem_c, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(tmem_c), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(tmem_c), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
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
// The feeding and issuing warps walk along as a whole and one lane issues: what comes before is then the same in every lane for
// all the compiler knows, and addresses and descriptors are made in uniform registers, where the instructions take them.  (From
// one lane's own registers a stage of one block cost 300 ns beside its copies and MMAs.)
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}\n" : "=r"(is));
  return is != 0;
}
__device__ __forceinline__ int same_in_warp(int v) { return __shfl_sync(0xffffffffu, v, 0); }
template <bool CLUSTER> __device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, int* err) {
  const bool mine = CLUSTER ? mbar_wait_cluster(bar, parity, err) : mbar_wait(bar, parity, err);
  return __all_sync(0xffffffffu, mine ? 1 : 0) != 0;
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

template <typename T> __device__ __forceinline__ uint4 pack16(const float* y);
template <> __device__ __forceinline__ uint4 pack16<float>(const float* y) {
  return make_uint4(__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3]));
}
template <> __device__ __forceinline__ uint4 pack16<__nv_bfloat16>(const float* y) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&p);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Four sums with the token's scale, the channels' and their bias.
__device__ __forceinline__ void scaled4(const int* sum, float s, float4 c, float4 b, float* y) {
  y[0] = fmaf(static_cast<float>(sum[0]), s * c.x, b.x);
  y[1] = fmaf(static_cast<float>(sum[1]), s * c.y, b.y);
  y[2] = fmaf(static_cast<float>(sum[2]), s * c.z, b.z);
  y[3] = fmaf(static_cast<float>(sum[3]), s * c.w, b.w);
}

// Where 16 bytes of a turned row lie, so that neither eight rows' same piece nor a row's pieces share banks.
template <typename T> __device__ __forceinline__ int turned(int row, int piece) {
  if constexpr (sizeof(T) == 4) return row * 128 + ((piece ^ (row & 7)) * 16);
  else return row * 64 + ((piece ^ ((row >> 1) & 3)) * 16);
}

// Rows low .. high and the first `cols` columns of 32 x 32 turned results to where the first belongs, word by word of W, the loads
// of eight ahead of their stores.  (Rows off 16 bytes: 7,052 x 768 -> 3,252 bfloat16 in words of eight bytes 35.4 -> 22.0 us,
// -> 3,251 result by result 28.4, loads and stores in turn 35.4.  Words of two results gained nothing over single ones.)
template <typename W, typename T>
__device__ __forceinline__ void store_rows(const unsigned char* turn, T* out, int n, int low, int high, int cols) {
  constexpr int ACROSS = 32 * sizeof(T) / sizeof(W), ROWS = 32 / ACROSS;
  const int lane = threadIdx.x & 31, at = lane % ACROSS * static_cast<int>(sizeof(W) / sizeof(T)), byte = at * static_cast<int>(sizeof(T));
  if (at >= cols) return;
#pragma unroll 1
  for (int r0 = lane / ACROSS; r0 < high; r0 += 8 * ROWS) {
    W y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = *reinterpret_cast<const W*>(turn + turned<T>(r0 + i * ROWS, byte / 16) + byte % 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = r0 + i * ROWS;
      if (r >= low && r < high) *reinterpret_cast<W*>(out + static_cast<size_t>(r) * n + at) = y[i];
    }
  }
}

// SPLIT: CTAs that share a tile's k (1: none).  WHOLE (looked at without a split): pieces of 16 bytes of the result lie at multiples of
// 16 bytes.  (Both kinds of store in one kernel cost whole results 4 %.)
template <typename T, int MODE, int CG, int SPLIT, bool WHOLE>
__global__ void __launch_bounds__(THREADS, 1)
product_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap wmap, const Int8ProductParams P, const Plan plan) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stages = plan.stages, stage_bytes = plan.stage_bytes, sub = plan.sub, a_bytes = plan.box * BK;
  const int bn = plan.bn, out_cols = MODE == INT8_GLU ? bn / 2 : bn;      // (columns of the result a tile)
  const int w_rows = bn / CG, w_bytes = w_rows * BK;                 // weight rows that this CTA fetches a tile
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + stages * stage_bytes);
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* acc_full = empty + MAX_STAGES;      // [2]
  uint64_t* acc_empty = acc_full + 2;           // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  unsigned char* turn = reinterpret_cast<unsigned char*>(tmem_slot + 4);
  float* scales = reinterpret_cast<float*>(turn + turn_bytes<T>());

  const int warp = same_in_warp(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rank = CG == 2 || SPLIT > 1 ? same_in_warp(static_cast<int>(cluster_rank())) : 0;
  const int m_tiles = (P.tokens + CG * BM - 1) / (CG * BM), n_tiles = (P.n + out_cols - 1) / out_cols, tiles = m_tiles * n_tiles;
  const int all_kb = (P.k + BK - 1) / BK;
  const int kb0 = SPLIT > 1 ? rank * all_kb / SPLIT : 0, kb1 = SPLIT > 1 ? (rank + 1) * all_kb / SPLIT : all_kb;
  const int first = blockIdx.x / (SPLIT * CG), step = gridDim.x / (SPLIT * CG);

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(full + s, 2); mbar_init(empty + s, 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(acc_full + a, 1); mbar_init(acc_empty + a, EPI_WARPS * CG); }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 1) {                                                              // the whole warp allocates tensor memory
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)), "r"(2 * ACC) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)), "r"(2 * ACC) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();                                                  // the pair's barriers exist
  tc_fence_after();
  const uint32_t tmem_base = same_in_warp(*tmem_slot);
  pdl_launch_dependents();

  // the weight rows of a tile that this CTA fetches (gate and up rows: two boxes, or one each of a pair's CTAs), and its
  // tokens: the tile's, and where they are fetched
  constexpr int BOXES = MODE == INT8_GLU && CG == 1 ? 2 : 1;
  auto weight_row = [&](int n, int box) {
    if (MODE == INT8_GLU) return ((CG == 2 ? rank : box) ? P.n : 0) + n * out_cols;
    return n * out_cols + (CG == 2 ? rank * w_rows : 0);
  };
  auto first_token = [&](int m) { return (m * CG + (CG == 2 ? rank : 0)) * BM; };
  auto first_fetched = [&](int m) { return P.tokens >= BM ? min(first_token(m), P.tokens - BM) : 0; };

  // SPLIT: what this CTA finishes of the cluster's tile (its share of the columns, of gate and up each half, and the tokens)
  int m0 = 0, n0 = 0;
  if (SPLIT > 1) tile_at(first, m_tiles, n_tiles, m0, n0);
  const int width = bn / SPLIT, half = out_cols, own = MODE == INT8_GLU ? width / 2 : width, own0 = n0 * out_cols + rank * own;
  const int row0 = first_fetched(m0), low = first_token(m0) - row0, high = min(BM, P.tokens - row0), quad_ints = plan.box * 4;
  float* token_scale = scales + 512;            // behind [gate, up][scale, bias][128]

  // A stage holds the tokens of its blocks of k, then the weights of them.
  auto feed = [&](auto of_weights) {
    constexpr bool WEIGHTS = decltype(of_weights)::value;
    const int block_bytes = WEIGHTS ? w_bytes : a_bytes;
    int m, n;
    if (WEIGHTS && first < tiles) {
      // The first weights start for the second-level cache before the dependency wait; nothing is read before it.
      tile_at(first, m_tiles, n_tiles, m, n);
      if (elect_one())
        for (int kb = kb0; kb < kb1 && kb < kb0 + stages * sub; ++kb)
          for (int box = 0; box < BOXES; ++box) tma_prefetch(&wmap, kb * BK, weight_row(n, box));
      __syncwarp();
    }
    pdl_wait();
    int s = 0, use = 0;                                                         // the ring's place, and how often it was filled
    bool ok = true;
    for (int tile = first; tile < tiles && ok; tile += step) {
      tile_at(tile, m_tiles, n_tiles, m, n);
      const int row = WEIGHTS ? weight_row(n, 0) : first_fetched(m);
      for (int kb = kb0; kb < kb1; kb += sub) {
        if (use > 0 && !mbar_wait_warp<false>(empty + s, (use - 1) & 1, P.err)) { ok = false; break; }
        const int blocks = min(sub, kb1 - kb);
        unsigned char* st = ring + s * stage_bytes + (WEIGHTS ? sub * a_bytes : 0);
        const uint32_t bar = CG == 2 ? cta_address(full + s, 0) : smem_u32(full + s);
        if (elect_one()) {
          if (CG == 1 || rank == 0) mbar_expect_tx(full + s, CG * blocks * block_bytes);
          for (int j = 0; j < blocks; ++j, st += block_bytes) {
            tma_load<CG>(st, WEIGHTS ? &wmap : &qmap, (kb + j) * BK, row, bar);
            if (WEIGHTS && BOXES == 2) tma_load<CG>(st + w_bytes / 2, &wmap, (kb + j) * BK, weight_row(n, 1), bar);
          }
        }
        __syncwarp();
        if (++s == stages) { s = 0; ++use; }
      }
    }
  };
  if (warp == 0) {
    feed(std::true_type());
  } else if (warp == 2 + EPI_WARPS) {
    feed(std::false_type());
  } else if (warp == 1) {
    pdl_wait();
    if (CG == 1 || rank == 0) {
      const uint32_t idesc = instr_desc<CG>(bn);
      const uint64_t da = smem_desc(smem_u32(ring)), db = smem_desc(smem_u32(ring + sub * a_bytes));
      int s = 0, use = 0, local = 0;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += step, ++local) {
        const int acc = local & 1, turns = local >> 1;
        if (turns > 0) ok = mbar_wait_warp<CG == 2>(acc_empty + acc, (turns - 1) & 1, P.err);       // the epilogues have read this accumulator
        if (!ok) break;
        tc_fence_after();
        const uint32_t tmem_c = tmem_base + acc * ACC;
        for (int kb = kb0; kb < kb1; kb += sub) {
          ok = mbar_wait_warp<false>(full + s, use & 1, P.err);
          if (!ok) break;
          tc_fence_after();
          const int blocks = min(sub, kb1 - kb);
          uint64_t a = da + static_cast<uint32_t>(s * stage_bytes >> 4), b = db + static_cast<uint32_t>(s * stage_bytes >> 4);
          if (elect_one()) {
            for (int j = 0; j < blocks; ++j, a += static_cast<uint32_t>(a_bytes >> 4), b += static_cast<uint32_t>(w_bytes >> 4))
#pragma unroll
              for (int k = 0; k < BK / 32; ++k) mma_i8<CG>(tmem_c, a + k * 2, b + k * 2, idesc, (kb > kb0 || j > 0 || k > 0) ? 1u : 0u);
            mma_commit<CG>(empty + s);                                          // the stage is free when these MMAs have read it
          }
          __syncwarp();
          if (++s == stages) { s = 0; ++use; }
        }
        if (elect_one()) mma_commit<CG>(acc_full + acc);                        // the tile's sums are complete
        __syncwarp();
      }
    }
  } else if (SPLIT == 1) {
    pdl_wait();
    const int quarter = warp & 3, part = (warp - 2) >> 2;
    constexpr int ROW = 32 * sizeof(T);                                         // bytes of a turned row
    unsigned char* mine = turn + (warp - 2) * (32 * ROW);
    float* sc = scales + (warp - 2) * (SCALES / 4 / EPI_WARPS);
    constexpr int HALVES = MODE == INT8_GLU ? 2 : 1;
    int local = 0;
    T* out = static_cast<T*>(P.out);
    constexpr int LANES = 32 * sizeof(T) / 16;                                  // lanes that a row's 32 results take, 16 bytes each
    // scales and bias of a tile's columns (and the token's scale) come from memory while the tile before is worked on
    constexpr int PIECES = ACC / HALVES / 32 / PARTS;                           // of 32 columns, at most
    float c_next[PIECES][HALVES], b_next[PIECES][HALVES], s_next = 0.0f;
    auto fetch = [&](int tile) {
      int m, n;
      tile_at(tile, m_tiles, n_tiles, m, n);
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          const int in = (part + i * PARTS) * 32 + lane, col = n * out_cols + in;
          const bool there = in < out_cols && col < P.n;
          c_next[i][h] = there ? P.c[h * P.n + col] : 0.0f;
          b_next[i][h] = there && P.bias ? P.bias[h * P.n + col] : 0.0f;
        }
      const int row = first_fetched(m) + quarter * 32 + lane;
      s_next = row < P.tokens ? P.s[row] : 0.0f;
    };
    if (first < tiles) fetch(first);
    for (int tile = first; tile < tiles; tile += step, ++local) {
      int m, n;
      tile_at(tile, m_tiles, n_tiles, m, n);
      const int acc = local & 1;
      const int row0 = first_fetched(m) + quarter * 32;
      const int low = max(0, first_token(m) - row0), high = min(32, P.tokens - row0);       // the rows of these 32 that are stored
      __syncwarp();
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          sc[(i * HALVES + h) * 64 + lane] = c_next[i][h];
          sc[(i * HALVES + h) * 64 + 32 + lane] = b_next[i][h];
        }
      const float s = s_next;
      if (tile + step < tiles) fetch(tile + step);
      __syncwarp();
      if (!mbar_wait(acc_full + acc, (local >> 1) & 1, P.err)) break;
      tc_fence_after();
      const uint32_t base = tmem_base + acc * ACC + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
      for (int p = part, i = 0; p * 32 < out_cols; p += PARTS, ++i) {
        const int col0 = n * out_cols + p * 32, cols = min(min(32, out_cols - p * 32), P.n - col0);
        if (high <= low || cols <= 0) break;                                    // (the whole warp)
        int g[32], u[MODE == INT8_GLU ? 32 : 1];
        tmem_ld32(base + p * 32, g);
        if constexpr (MODE == INT8_GLU) tmem_ld32(base + out_cols + p * 32, u);
        tmem_ld_wait();
        const float4* gs = reinterpret_cast<const float4*>(sc + i * HALVES * 64);
        uint4 packed[LANES];                                                    // (all of them before the first store: the scales' loads pass no store)
#pragma unroll
        for (int e = 0; e < LANES; ++e) {
          constexpr int N = 16 / sizeof(T);
          float y[N];
#pragma unroll
          for (int z = 0; z < N; z += 4) {
            const int at = e * N + z;
            scaled4(g + at, s, gs[at / 4], P.bias ? gs[8 + at / 4] : make_float4(0.0f, 0.0f, 0.0f, 0.0f), y + z);
            if constexpr (MODE == INT8_GLU) {
              float up[4];
              scaled4(u + at, s, gs[16 + at / 4], P.bias ? gs[24 + at / 4] : make_float4(0.0f, 0.0f, 0.0f, 0.0f), up);
#pragma unroll
              for (int j = 0; j < 4; ++j) y[z + j] = gate_up<sizeof(T) == 4>(y[z + j], up[j], P.limit, P.alpha);
            }
          }
          packed[e] = pack16<T>(y);
        }
#pragma unroll
        for (int e = 0; e < LANES; ++e) *reinterpret_cast<uint4*>(mine + turned<T>(lane, e)) = packed[e];
        __syncwarp();
        T* to = out + static_cast<size_t>(row0) * P.n + col0;
        if constexpr (WHOLE && sizeof(T) == 2) {                                // (whole pieces of 16 bytes, up to the last column too)
#pragma unroll
          for (int q = 0; q < LANES; ++q) {
            const int r = q * (32 / LANES) + lane / LANES, chunk = lane % LANES;
            if (r >= low && r < high && chunk * 8 < cols)
              *reinterpret_cast<uint4*>(to + static_cast<size_t>(r) * P.n + chunk * 8) = *reinterpret_cast<const uint4*>(mine + turned<T>(r, chunk));
          }
        } else if constexpr (WHOLE) {
          store_rows<uint4, T>(mine, to, P.n, low, high, cols);
        } else if (sizeof(T) == 2 && ((reinterpret_cast<uintptr_t>(to) / 2 | P.n | cols) & 3) == 0) {
          store_rows<uint2, T>(mine, to, P.n, low, high, cols);
        } else {
          store_rows<T, T>(mine, to, P.n, low, high, cols);
        }
        __syncwarp();
      }
      tc_fence_before();                                                        // the loads of this accumulator are done
      __syncwarp();
      if (lane == 0) mbar_hand_back<CG>(acc_empty + acc);
    }
  } else {
    // One tile a cluster: scales and bias of the columns that this CTA will finish, then the tokens' scales.
    pdl_wait();
    for (int i = threadIdx.x - 64; i < own; i += 32 * EPI_WARPS)
#pragma unroll
      for (int h = 0; h < (MODE == INT8_GLU ? 2 : 1); ++h) {
        const bool in = own0 + i < P.n;
        scales[h * 256 + i] = in ? P.c[h * P.n + own0 + i] : 0.0f;
        scales[h * 256 + 128 + i] = in && P.bias ? P.bias[h * P.n + own0 + i] : 0.0f;
      }
    for (int i = threadIdx.x - 64; i < high; i += 32 * EPI_WARPS) token_scale[i] = P.s[row0 + i];
    if (first < tiles) mbar_wait(acc_full, 0, P.err);
    tc_fence_after();
  }

  if constexpr (SPLIT > 1) {
    // Everybody's MMAs have read their rings, which take the others' sums now: [from][columns / 4][tokens of the box][4].
    int* sums = reinterpret_cast<int*>(ring);
    __syncwarp();
    cluster_sync();
    if (warp >= 2 && warp < 2 + EPI_WARPS) {
      const int row = (warp & 3) * 32 + lane;
      if ((warp & 3) * 32 < high) {
        const uint32_t base = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
#pragma unroll 1
        for (int c = ((warp - 2) >> 2) * 32; c < bn; c += PARTS * 32) {
          int v[32];
          tmem_ld32(base + c, v);
          tmem_ld_wait();
          int up = MODE == INT8_GLU && c >= half ? own : 0, to = (c - (up ? half : 0)) / own, at = c - (up ? half : 0) - to * own;
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            if (c + e < bn && row < high) {
              const uint32_t dst = cta_address(sums + (rank * (width / 4) + (up + at) / 4) * quad_ints + row * 4, to);
              asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(dst), "r"(v[e]), "r"(v[e + 1]), "r"(v[e + 2]), "r"(v[e + 3]) : "memory");
            }
            if ((at += 4) == own) {
              at = 0;
              if (++to == SPLIT) { to = 0; up = own; }
            }
          }
        }
      }
    }
    __syncwarp();
    cluster_sync();
    // A warp takes 8 tokens x 16 columns at a time: a lane four columns of a token.
    T* out = static_cast<T*>(P.out);
    const bool whole = (reinterpret_cast<uintptr_t>(out) | (static_cast<size_t>(P.n) * sizeof(T))) % (4 * sizeof(T)) == 0;
    const int quads = own / 4, across = (quads + 3) / 4, blocks = (high - low + 7) / 8 * across;
    for (int i = warp; i < blocks; i += THREADS / 32) {
      const int row = low + i / across * 8 + (lane & 7), quad = i % across * 4 + (lane >> 3), col = own0 + quad * 4;
      if (row >= high || quad >= quads || col >= P.n) continue;
      float y[2][4];
#pragma unroll
      for (int h = 0; h < (MODE == INT8_GLU ? 2 : 1); ++h) {
        int t[4] = {0, 0, 0, 0};
#pragma unroll
        for (int from = 0; from < SPLIT; ++from) {
          const int4 v = *reinterpret_cast<const int4*>(sums + (from * (width / 4) + h * quads + quad) * quad_ints + row * 4);
          t[0] += v.x; t[1] += v.y; t[2] += v.z; t[3] += v.w;
        }
        scaled4(t, token_scale[row], *reinterpret_cast<const float4*>(scales + h * 256 + quad * 4),
                *reinterpret_cast<const float4*>(scales + h * 256 + 128 + quad * 4), y[h]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (MODE == INT8_GLU) y[0][e] = gate_up<sizeof(T) == 4>(y[0][e], y[1][e], P.limit, P.alpha);
      T* dst = out + static_cast<size_t>(row0 + row) * P.n + col;
      if (whole && col + 4 <= P.n) {
        __align__(16) T r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = from_f32<T>(y[0][e]);
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(r);
        else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(r);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < P.n) dst[e] = from_f32<T>(y[0][e]);
      }
    }
  }
  // Everybody meets here on every path; then the allocating warp gives the tensor memory back.
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  if (CG == 2) cluster_sync();                                                  // (the pair's MMAs and arrivals are over)
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(2 * ACC) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(2 * ACC) : "memory");
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

template <typename T, int MODE, int CG, int SPLIT, bool WHOLE>
static int launch(const Int8ProductParams& P, const Plan& plan, int blocks, int cluster, const Int8Device& device, cudaStream_t stream) {
  static bool set[64];
  int rc = int8_launch_limit(product_kernel<T, MODE, CG, SPLIT, WHOLE>, SMEM_MOST, device, set);
  if (rc != 0) return rc;
  CUtensorMap qmap, wmap;
  rc = tensor_map(&qmap, P.q, P.tokens, P.k, P.q_pitch, plan.box);
  if (rc == 0) rc = tensor_map(&wmap, P.w, static_cast<long long>(P.n) * (MODE == INT8_GLU ? 2 : 1), P.k, P.w_pitch,
                                 CG == 2 || MODE == INT8_GLU ? plan.bn / 2 : plan.bn);
  if (rc != 0) return rc;
  return b200_launch(product_kernel<T, MODE, CG, SPLIT, WHOLE>, dim3(blocks), dim3(THREADS), smem_fixed<T>() + plan.stages * plan.stage_bytes, stream,
                     cluster, qmap, wmap, P, plan);
}

// Stages of as much k as leaves the ring four of them: a stage costs the threads that feed and issue about 190 ns beside its
// copies and MMAs (300 ns with one block of k and few columns).
static void set_stages(Plan& p, int rows_a_cta, int fixed) {
  const int block = (p.box + rows_a_cta) * BK, room = SMEM_MOST - fixed;
  p.sub = p.way == 0 ? 1 : room / (4 * block);
  if (p.sub < 1) p.sub = 1;
  if (p.sub > 4) p.sub = 4;
  p.stage_bytes = p.sub * block;
  p.stages = room / p.stage_bytes;
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
}

// How a product is cut up (see the top of the file): the way that takes its fullest SM the least, by a model of it in us.  `quads`:
// clusters of four CTAs that run side by side.
//   a block of k      what its bytes take at 126 GB/s an SM, 0.19 us at least (a pair's: or its MMAs' time)
//   a tile's epilogue 0.0024 us a column, 0.4 us more where warps find pieces of less than 32 columns; it hides behind the next tile
//   the weights       no less than at 8.4 TB/s (a part of them comes while the rows go to 8 bits)
//   sharing k         1.4 us with two CTAs, 3.8 us with four (with the cluster's launch; the exchange itself is below 1 us)
// Fitted to 140 products of 20 to 2,048 tokens that were run all ways (behind rows to 8 bits, cold weights): the way chosen takes 1.6 %
// longer than the best one on average.  (Of it, 64 columns / 128 / 32 in two rounds, 64 tokens, 4,096 k, 6,144 columns: 9.5 / 11.9 /
// 12.0 us; 100 tokens, 12,288 k, 4,096 columns: 128 columns shared by four 16.1, 64 by two 16.6, 32 by none 18.9, pairs of 190 tokens
// 26.9 us at 24,576 gated columns where single tiles take 30.6.)
static inline Plan make_plan(int tokens, int n, int k, int mode, int sms, int quads, int fixed) {
  Plan p = {};
  const int glu = mode == INT8_GLU ? 2 : 1, kb = (k + BK - 1) / BK;
  const long long cols = static_cast<long long>(n) * glu, m_tiles = (tokens + BM - 1) / BM;
  p.box = tokens >= BM ? BM : (tokens + 7) / 8 * 8;
  const double memory = static_cast<double>(cols) * k / 8.4e6;
  double best = 0.0;
  auto consider = [&](int way, int bn, long long tiles, long long side_by_side, double block, int blocks, double more) {
    const long long rounds = (tiles + side_by_side - 1) / side_by_side;
    const double products = blocks * block, epilogue = 0.0024 * bn + (bn / glu % 32 ? 0.4 : 0.0);
    const double all = products * (way > 1 ? rounds : 1) + (way > 1 ? 0.0 : (rounds - 1) * (products > epilogue ? products : epilogue));
    const double cost = (all > memory ? all : memory) + (way > 1 ? rounds * (epilogue / 2 + more) : epilogue + more);
    if (best == 0.0 || cost < best) { best = cost; p.way = way; p.bn = bn; }
  };
  for (int split = 1; split <= 4 && split <= kb; split *= 2)
    for (int bn = 256; bn >= 32; bn -= bn > 128 ? 32 : 16) {
      if (bn % (4 * glu * split) != 0) continue;
      const double block = (p.box + bn) * BK / 126e3;
      consider(split, bn, m_tiles * ((cols + bn - 1) / bn), split == 1 ? sms : split == 2 ? sms / 2 : quads, block > 0.19 ? block : 0.19,
               (kb + split - 1) / split, split == 1 ? 0.0 : split == 2 ? 1.4 : 3.8);
    }
  if (tokens > BM)
    for (int bn = 256; bn >= 128; bn -= 32) {
      const double bytes = (BM + bn / 2) * BK / 126e3, mma = bn * 0.0011;
      consider(0, bn, (tokens + 255ll) / 256 * ((cols + bn - 1) / bn), sms / 2, bytes > mma ? bytes : mma, kb, 0.12);
    }
  set_stages(p, p.way == 0 ? p.bn / 2 : p.bn, fixed);
  return p;
}

// Clusters of four CTAs of the split kernel that run side by side (1 where the device does not say).
template <typename T, int MODE> static int quads_side_by_side(int device) {
  static int known[64];                        // plus one, of the devices that were asked
  if (device < 0 || device >= 64) return 1;
  if (known[device] == 0) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(4);
    config.blockDim = dim3(THREADS);
    config.dynamicSmemBytes = SMEM_MOST;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 4;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(product_kernel<T, MODE, 1, 4, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MOST) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, product_kernel<T, MODE, 1, 4, true>, &config) != cudaSuccess || n < 1)
      n = 1;
    known[device] = n + 1;
  }
  return known[device] - 1;
}

template <typename T, int MODE> static int product(const Int8ProductParams& P, const Int8Device& device, cudaStream_t stream) {
  const int sms = device.sms;
  const Plan plan = make_plan(P.tokens, P.n, P.k, MODE, sms, quads_side_by_side<T, MODE>(device.index), smem_fixed<T>());
  const int tall = plan.way == 0 ? 2 * BM : BM, wide = plan.bn / (MODE == INT8_GLU ? 2 : 1);
  const long long tiles = static_cast<long long>((P.tokens + tall - 1) / tall) * ((P.n + wide - 1) / wide);
  if (tiles > 0x0fffffff || plan.stages < 2) return B200_BAD_SIZE;
  const int t = static_cast<int>(tiles);
  const bool whole = (reinterpret_cast<uintptr_t>(P.out) | (static_cast<size_t>(P.n) * sizeof(T)) | (wide * sizeof(T))) % 16 == 0;
  const int pairs = 2 * (t < sms / 2 ? t : sms / 2), ctas = t < sms ? t : sms;
  if (plan.way == 0) return whole ? launch<T, MODE, 2, 1, true>(P, plan, pairs, 2, device, stream) : launch<T, MODE, 2, 1, false>(P, plan, pairs, 2, device, stream);
  if (plan.way == 1) return whole ? launch<T, MODE, 1, 1, true>(P, plan, ctas, 0, device, stream) : launch<T, MODE, 1, 1, false>(P, plan, ctas, 0, device, stream);
  return plan.way == 2 ? launch<T, MODE, 1, 2, true>(P, plan, 2 * t, 2, device, stream) : launch<T, MODE, 1, 4, true>(P, plan, 4 * t, 4, device, stream);
}

}  // namespace i8tc
