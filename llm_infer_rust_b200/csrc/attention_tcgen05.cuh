// What the tcgen05 attention kernels (attention_tcgen05.cu, prefix_tcgen05.cu) have in common, head size 128: instructions and
// descriptors, and what a softmax thread does with its row of a block.
#pragma once
#include <cuda.h>
#include <math.h>
#include <string.h>

#include "common.cuh"
#include "pairs.cuh"

typedef __nv_bfloat16 bf16;
constexpr int D = 128;
constexpr int BQ = 128;                  // query vectors per CTA
constexpr int BKV = 128;                 // keys per block
constexpr int HALF = BKV * 128;          // bytes of a [128 rows x 64 columns] half tile
constexpr int TILE = 2 * HALF;           // bytes of a [128 x 128] bfloat16 tile
constexpr int TMEM_COLS = 512;           // S buffers (and P in their first 64 columns): columns 0..127 and 128..255; O: 256..383
constexpr int TBL_ENTRIES = 2048;         // page numbers of a row that the copy warp keeps in shared memory (the rest it reads as before)
constexpr float RESCALE_STEP = 8.0f;     // the reference maximum follows only growth beyond 2^8

__device__ __forceinline__ void mbar_init(uint64_t* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
// All lanes of a warp wait and agree on the outcome: the collective tensor-memory loads that follow need the
// warp whole, also when a wait has run out.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, int* err) {
  const bool mine = mbar_wait(bar, parity, err);
  return __all_sync(0xffffffffu, mine ? 1 : 0) != 0;
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n"
               ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y) : "memory");
}
// K-major tile in the 128-byte swizzle: 8-row groups 1024 bytes apart, leading byte offset unused (1).
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
  const uint32_t lo = ((addr >> 4) & 0x3FFFu) | (1u << 16);
  const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}
// MN-major tile in the 128-byte swizzle (rows = k, 64 MN elements = 128 bytes contiguous): 8-row groups 1024 bytes
// apart (stride byte offset), the next 64 MN elements HALF bytes further (leading byte offset).
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr) {
  const uint32_t lo = ((addr >> 4) & 0x3FFFu) | (static_cast<uint32_t>(HALF >> 4) << 16);
  const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}
// float accumulator, bfloat16 operands, M 128, N 128; B is K-major for S = Q K^T and MN-major for P V.
constexpr uint32_t kDescQK = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t kDescPV = kDescQK | (1u << 16);

__device__ __forceinline__ void umma(uint32_t tmem_c, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
               ::"r"(tmem_c), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
// The A operand from tensor memory: 16-bit elements packed two to a column (k = 2c, 2c + 1 in column c of lane m).
__device__ __forceinline__ void umma_a_tmem(uint32_t tmem_c, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
               ::"r"(tmem_c), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
// True in one lane of a whole warp.  The warp that issues products walks along as a whole and only the instruction itself is one
// lane's: what comes before it is then the same in every lane for all the compiler knows, and descriptors are made in uniform
// registers, where the instruction takes them.  (From one lane's own registers a product took 100 cycles to issue, so 35: 8,192 tokens x
// 16 heads 299 -> 275 us.)
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}\n" : "=r"(is));
  return is != 0;
}
__device__ __forceinline__ int same_in_warp(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
               "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                 "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                 "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// 64 consecutive columns of this thread's lane, in one load and one wait.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&v)[64]) {
  uint32_t r[64];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n"
               "tcgen05.wait::ld.sync.aligned;\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
               : "r"(taddr) : "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float (&v)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
               "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
               "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n"
               ::"r"(taddr), "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
                 "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])),
                 "r"(__float_as_uint(v[8])), "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])), "r"(__float_as_uint(v[11])),
                 "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])), "r"(__float_as_uint(v[14])), "r"(__float_as_uint(v[15])),
                 "r"(__float_as_uint(v[16])), "r"(__float_as_uint(v[17])), "r"(__float_as_uint(v[18])), "r"(__float_as_uint(v[19])),
                 "r"(__float_as_uint(v[20])), "r"(__float_as_uint(v[21])), "r"(__float_as_uint(v[22])), "r"(__float_as_uint(v[23])),
                 "r"(__float_as_uint(v[24])), "r"(__float_as_uint(v[25])), "r"(__float_as_uint(v[26])), "r"(__float_as_uint(v[27])),
                 "r"(__float_as_uint(v[28])), "r"(__float_as_uint(v[29])), "r"(__float_as_uint(v[30])), "r"(__float_as_uint(v[31]))
               : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
}
// 32 columns of this thread's lane from 32 registers; the caller waits (tcgen05.wait::st) before it tells anyone.
__device__ __forceinline__ void tmem_st32_raw(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
               "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
               "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                 "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
                 "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
                 "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
               "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                 "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
               "tcgen05.wait::ld.sync.aligned;\n"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                 "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ float fast_exp2(float x) {      // 2^x, one special-function instruction (-inf gives 0)
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

// Byte offset of (row r, 16-byte chunk c of 16) inside a [128 x 128] bfloat16 tile of two swizzled halves.
__device__ __forceinline__ int swz(int r, int c) { return (c >> 3) * HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4); }

// ---------------------------------------------------------------------------------------------------------------
// What the softmax threads of both kernels do.  A thread owns one query row: lane r of tensor memory.

// The row's Q vector into its K-major tile in the 128-byte swizzle (zeros for a row that is not used), chunks
// c_lo .. c_lo + CHUNKS - 1 of 16.
template <int CHUNKS>
__device__ __forceinline__ void write_q_row(unsigned char* q_tile, const bf16* src, int r, bool used, int c_lo) {
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    const int c = c_lo + i;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (used) v = *reinterpret_cast<const uint4*>(src + c * 8);
    *reinterpret_cast<uint4*>(q_tile + swz(r, c)) = v;
  }
  proxy_fence();
}

// Row r of an MN-major value tile (128 dims in two halves of 128 bytes), chunks c_lo .. c_lo + CHUNKS - 1 of 16 set to zero.
template <int CHUNKS>
__device__ __forceinline__ void zero_value_row(unsigned char* v_tile, int r, int c_lo) {
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (int c = c_lo; c < c_lo + CHUNKS; ++c) *reinterpret_cast<uint4*>(v_tile + (c >> 3) * HALF + r * 128 + (c & 7) * 16) = zero;
}

struct RowState {
  float m_ref = -INFINITY;     // reference maximum (log2 units): follows the row's maximum in steps of RESCALE_STEP
  float l_run = 0.0f;          // sum of the probabilities relative to it
};

// One block of 128 keys for this thread's row.  The scores lie in the 128 columns from s_base on; the bfloat16
// probabilities go back over the first 64 of them, two to a column (the A operand of P V), and are in tensor memory
// when the function returns.  The row sees keys lo_key .. hi_key (none: hi_key -1).  `block` counts the row's blocks from 0; P V of block - 1 commits to `pv_done`.  Every
// phase of that barrier is waited for here, in order: before the accumulator at o_base is rescaled (the row's
// maximum grew by more than the step), else at the end, when that product has long finished.  A wait by parity
// cannot tell "phase b - 1 is not finished" from "phase b - 2 is not finished": a waiter that skipped a phase
// would pass at once.  Returns false when a wait ran out.
__device__ __forceinline__ bool softmax_block(uint32_t s_base, uint32_t o_base, int first_key, int lo_key, int hi_key,
                                              bool masked, float scale_log2, int block, uint64_t* pv_done, RowState& st,
                                              int* err) {
  tc_fence_after();
  // pass 1: the row's maximum over the block's visible keys (of the raw scores; the scale is positive)
  float mx = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 2; ++c) {
    float v[64];
    tmem_ld64(s_base + c * 64, v);
    if (masked) {
#pragma unroll
      for (int e = 0; e < 64; ++e) {
        const int key = first_key + c * 64 + e;
        const bool vis = key >= lo_key && key <= hi_key;
        mx = fmaxf(mx, vis ? v[e] : -INFINITY);
      }
    } else {
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};      // four chains instead of one
#pragma unroll
      for (int e = 0; e < 64; e += 4) {
        m4[0] = fmaxf(m4[0], v[e]); m4[1] = fmaxf(m4[1], v[e + 1]); m4[2] = fmaxf(m4[2], v[e + 2]); m4[3] = fmaxf(m4[3], v[e + 3]);
      }
      mx = fmaxf(mx, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
    }
  }
  mx = hi_key >= 0 ? mx * scale_log2 : -INFINITY;
  // The reference follows the maximum when it grew by more than the step (or there was none yet).
  const bool raise = mx > st.m_ref + RESCALE_STEP || (st.m_ref == -INFINITY && mx > -INFINITY);
  const float m_new = raise ? mx : st.m_ref;
  const float corr = raise ? (st.m_ref == -INFINITY ? 0.0f : exp2f(st.m_ref - m_new)) : 1.0f;
  const float base = m_new == -INFINITY ? 0.0f : m_new;
  bool pv_seen = block == 0;
  // The accumulator may be rescaled only between two products: P V of the block before has to be finished.
  if (block > 0 && __any_sync(0xffffffffu, raise ? 1 : 0)) {
    if (!mbar_wait_warp(pv_done, (block - 1) & 1, err)) return false;
    pv_seen = true;
    tc_fence_after();
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
      float o[32];
      tmem_ld32(o_base + c * 32, o);
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] *= corr;
      tmem_st32(o_base + c * 32, o);
    }
  }
  st.l_run = st.l_run * corr;
  st.m_ref = m_new;
  // pass 2: probabilities relative to the reference and their sum; those of columns 64c .. 64c + 63 go back into
  // tensor memory over the scores that were just read (columns 32c .. 32c + 31)
  const float neg_base = hi_key >= 0 ? -base : -INFINITY;      // a row that is not used gets zeros
  float sum4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
  for (int c = 0; c < 2; ++c) {
    float v[64];
    tmem_ld64(s_base + c * 64, v);
    if (masked) {
#pragma unroll
      for (int e = 0; e < 64; ++e) {
        const int key = first_key + c * 64 + e;
        const bool vis = key >= lo_key && key <= hi_key;
        v[e] = vis ? fast_exp2(fmaf(v[e], scale_log2, neg_base)) : 0.0f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 64; ++e) v[e] = fast_exp2(fmaf(v[e], scale_log2, neg_base));
    }
    uint32_t pr[32];
#pragma unroll
    for (int e = 0; e < 64; e += 2) {
      sum4[(e >> 1) & 3] += v[e] + v[e + 1];
      __nv_bfloat162 two = __floats2bfloat162_rn(v[e], v[e + 1]);
      pr[e >> 1] = *reinterpret_cast<uint32_t*>(&two);
    }
    tmem_st32_raw(s_base + c * 32, pr);
  }
  st.l_run += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
  tmem_wait_st();                                      // P is in tensor memory
  return pv_seen || mbar_wait_warp(pv_done, (block - 1) & 1, err);
}

// The two-tile kernel's block: all 128 scores in registers (one load of the row, where softmax_block waits for four), and the
// products with the values begin when half of the weights stand: `half_done` is called behind the first 64 keys' weights.
// S of a block is issued behind P V of the block before it, so whoever has seen these scores may touch the accumulator:
// pv_done is not asked.  A tile walks a chain of its own latencies (measured with softmax_block, SM cycles a block at 8,192
// tokens: 2,040 until the next scores stand, 2,700 in the softmax, 1,720 of those behind the maximum, for 1,024 of
// special-function work), so what shortens the chain counts: 8,192 tokens x 16 heads 340 -> 302 us, 16,384 x 32 2,165 us
// (1,015 TFLOP/s).  Behind the maximum the thread's issue slots are the chain, so scale and sum take two scores an instruction
// (with the MMAs issued by a whole warp: 275 -> 265 us, 3,000 tokens 58.6 -> 56.8; from the two before both, 16,384 x 32 2,283 -> 2,171).
// The weights are added up as softmax_block adds them, a pair's two and then pairs into four sums, so that both kernels give the
// same bits: which of them runs follows from the other rows of the step.  (Every weight into a sum of its own place, one addition less
// in the chain, was 264 us.)  Two threads a row, which pay for the further forms below, were slower here (483 us: sixteen warps leave
// 96 registers a thread, so the scores are read twice).
__device__ __forceinline__ void tmem_ld32_begin(uint32_t taddr, float (&v)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
               "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
                 "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
                 "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
                 "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
               : "r"(taddr));
}
template <typename F>
__device__ __forceinline__ void softmax_row(uint32_t s_base, uint32_t o_base, int first_key, int lo_key, int hi_key, bool masked,
                                            float scale_log2, int block, RowState& st, const F& half_done) {
  tc_fence_after();
  float v[4][32];
#pragma unroll
  for (int c = 0; c < 4; ++c) tmem_ld32_begin(s_base + c * 32, v[c]);
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int e = 0; e < 32; ++e) asm volatile("" : "+f"(v[c][e]));      // (used only behind the wait)
  if (masked) {
    const int lo = lo_key - first_key, hi = hi_key - first_key;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int e = 0; e < 32; ++e) v[c][e] = c * 32 + e >= lo && c * 32 + e <= hi ? v[c][e] : -INFINITY;
  }
  float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int e = 0; e < 32; ++e) m4[e & 3] = fmaxf(m4[e & 3], v[c][e]);
  const float raw = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
  const float mx = hi_key >= 0 ? raw * scale_log2 : -INFINITY;
  const bool raise = mx > st.m_ref + RESCALE_STEP || (st.m_ref == -INFINITY && mx > -INFINITY);
  const float m_new = raise ? mx : st.m_ref;
  if (__any_sync(0xffffffffu, raise ? 1 : 0)) {
    const float corr = raise ? (st.m_ref == -INFINITY ? 0.0f : exp2f(st.m_ref - m_new)) : 1.0f;
    st.l_run *= corr;
    if (block > 0) {
#pragma unroll 1
      for (int c = 0; c < 8; ++c) {
        uint32_t o[16];
        tmem_ld16(o_base + c * 16, o);
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
        tmem_st16(o_base + c * 16, o);
      }
      tmem_wait_st();
    }
  }
  st.m_ref = m_new;
  const float neg_base = hi_key < 0 ? -INFINITY : m_new == -INFINITY ? 0.0f : -m_new;      // a row that is not used gets zeros
  f32x2 sums[2] = {0, 0};
  const f32x2 scale2 = twice(scale_log2), base2 = twice(neg_base);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t pr[16];
#pragma unroll
    for (int i = 0; i < 16; i += 2) {                  // two pairs of weights a turn: (a0, b0), (a1, b1)
      float a0, b0, a1, b1;
      unpack2(fma2(pack2(v[c][2 * i], v[c][2 * i + 1]), scale2, base2), a0, b0);
      unpack2(fma2(pack2(v[c][2 * i + 2], v[c][2 * i + 3]), scale2, base2), a1, b1);
      a0 = fast_exp2(a0);
      b0 = fast_exp2(b0);
      a1 = fast_exp2(a1);
      b1 = fast_exp2(b1);
      sums[(i >> 1) & 1] = add2(sums[(i >> 1) & 1], add2(pack2(a0, a1), pack2(b0, b1)));
      const __nv_bfloat162 p0 = __floats2bfloat162_rn(a0, b0), p1 = __floats2bfloat162_rn(a1, b1);
      pr[i] = *reinterpret_cast<const uint32_t*>(&p0);
      pr[i + 1] = *reinterpret_cast<const uint32_t*>(&p1);
    }
    tmem_st16(s_base + c * 16, pr);
    if (c == 1) {
      tmem_wait_st();
      half_done();
    }
  }
  float sum4[4];
  unpack2(sums[0], sum4[0], sum4[1]);
  unpack2(sums[1], sum4[2], sum4[3]);
  st.l_run += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
  tmem_wait_st();                                      // P is in tensor memory
}
