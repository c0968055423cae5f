// Products in 8-bit integers for a handful of tokens (decode steps): the weights are streamed by every thread for itself, no
// feeding thread and no barrier between copy and multiply; what it takes to bring the tokens to 8 bits runs in front.
//
//   weights   A thread of a warp (g = lane / 4, t = lane % 4) copies 16 bytes = 16 consecutive k of weight row g and of row
//             g + 8 (cp.async, past the first-level cache) into pieces of shared memory that are ITS OWN and reads them back
//             into the registers of the multiply: a step of 64 k.  DEPTH steps are on their way, 96 KB an SM.  mma.sync
//             m16n8k32 has the weight rows on its 16-row side and wants for thread t four k at 4 t and four at 16 + 4 t; a
//             sum over k does not care about the order of k, so the 16 bytes serve two instructions as they come, and the
//             tokens are read the same way.  (tcgen05 needs no faster rate here: 16 x 64 weights an SM every 44 cycles
//             are all that memory gives, two of these instructions.)
//   tokens    at most 8 a tile of the multiply, in shared memory for the whole kernel.  FUSED: they arrive as floats; 16
//             warps over the tokens (to a power of two) take each (behind the residual add and the norm) to 8 bits, in every CTA again: cheaper than
//             a kernel in front while a thread holds its share in registers (16,384 floats in all).
//   split     a CTA's 16 warps are WN groups of WK warps.  A group owns 16 weight rows at a time (INT8_GLU: 8 gate rows and the
//             same 8 up rows), its warps share k (warp s takes the steps s, s + WK, ...) and their sums meet in shared memory
//             (integers: any order); groups do not wait for one another, and the next rows' weights are on their way.
// One CTA an SM; rows are dealt out over all groups of all CTAs.  Before the dependency wait the first weights start for the
// second-level cache; nothing is read before it.
#pragma once
#include "int8_common.cuh"
#include "int8_rows.cuh"

namespace i8st {

constexpr int THREADS = 512, WARPS = 16, DEPTH = 6;
constexpr int RING = DEPTH * 2 * THREADS * 16;                   // 96 KB
constexpr int MOST_TOKENS = 16;
// What a launch may ask for: of the 227 KB of a block one is left to the arrays that the kernel declares itself.  takes() goes by it and
// the kernel's limit is set to it: a size above the limit would be refused at launch.
constexpr int DYNAMIC_MOST = 226 * 1024;

struct Plan {
  int wn, wk, steps;         // groups, shares of k, steps of 64 k a share
  int units, x_pitch;        // of 16 weight rows
};

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes that this thread's own copies brought (in order behind their wait).
__device__ __forceinline__ uint4 own_piece(const unsigned char* p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem_u32(p)) : "memory");
  return v;
}

// The tokens as floats to 8 bits in shared memory: 16 / T' warps a token (T' the power of two that holds them).
template <typename T, typename TG, bool NORM>
__device__ __forceinline__ void tokens_to_8_bits(const Int8RowsParams& R, int8_t* xs, int x_pitch, float* token_scale, float* sums, uint32_t* tops) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slots = R.tokens <= 1 ? 1 : R.tokens <= 2 ? 2 : R.tokens <= 4 ? 4 : 8, warps = WARPS / slots;
  const int token = warp / warps, threads = warps * 32, me = (warp % warps) * 32 + lane;
  const int chunks = x_pitch / 8;                                // (columns beyond k: zeros)
  const bool whole = R.whole != 0, here = token < R.tokens;
  float v[INT8_ROW_CHUNKS][8];
  float ss = 0.0f, most = 0.0f;
  if (here) {                                                    // (whole warps)
    const T* x = static_cast<const T*>(R.x) + static_cast<size_t>(token) * R.x_pitch;
    const T* residual = NORM && R.residual ? static_cast<const T*>(R.residual) + static_cast<size_t>(token) * R.k : nullptr;
    T* sum_out = NORM && R.sum_out && blockIdx.x == 0 ? static_cast<T*>(R.sum_out) + static_cast<size_t>(token) * R.k : nullptr;
    const TG* gain = static_cast<const TG*>(R.gain);
    Int8Raw<T> raw[INT8_ROW_CHUNKS], add[INT8_ROW_CHUNKS];
    Int8Raw<TG> g[INT8_ROW_CHUNKS];
#pragma unroll
    for (int i = 0; i < INT8_ROW_CHUNKS; ++i) {
      const int at = (me + i * threads) * 8;
      if (at >= R.k) continue;
      if (whole) {
        int8_load8<T, true>(x + at, 8, raw[i]);
        if (NORM && residual) int8_load8<T, true>(residual + at, 8, add[i]);
        if (NORM) int8_load8<TG, true>(gain + at, 8, g[i]);
      } else {
        int8_load8<T, false>(x + at, R.k - at, raw[i]);
        if (NORM && residual) int8_load8<T, false>(residual + at, R.k - at, add[i]);
        if (NORM) int8_load8<TG, false>(gain + at, R.k - at, g[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < INT8_ROW_CHUNKS; ++i) {
      const int at = (me + i * threads) * 8;
      if (at - lane * 8 >= R.k) continue;
      if (at < R.k) int8_sum<T>(raw[i], add[i], residual != nullptr, v[i]);
      if (NORM && sum_out) {
        if (!whole) int8_store8<T, false>(sum_out, at, R.k, v[i]);
        else if (at < R.k) int8_store8<T, true>(sum_out, at, R.k, v[i]);
      }
      if (at < R.k) int8_gain<TG, NORM, true>(g[i], v[i], at, R.k, ss, most);
    }
  }
  uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
  if (NORM) ss = warp_sum(ss);
  if (lane == 0) { tops[warp] = top; sums[warp] = ss; }
  __syncthreads();
  if (here) {
    top = 0u;
    ss = 0.0f;
    for (int w = token * warps; w < (token + 1) * warps; ++w) {
      top = max(top, tops[w]);
      ss += sums[w];
    }
    const Int8Step step = int8_step(top, NORM ? rsqrtf(ss / static_cast<float>(R.k) + R.eps) : 1.0f);
    if (me == 0) token_scale[token] = step.scale;
    int8_t* q = xs + token * x_pitch;
    for (int i = 0; me + i * threads < chunks; ++i) {
      const int at = (me + i * threads) * 8;
      uint2 b = make_uint2(0u, 0u);
#pragma unroll
      for (int j = 0; j < INT8_ROW_CHUNKS; ++j)
        if (j == i && at < R.k) b = make_uint2(int8_pack4(v[j], step), int8_pack4(v[j] + 4, step));
      *reinterpret_cast<uint2*>(q + at) = b;
    }
  }
}

// FUSED: the tokens are R's floats; else P.q, P.s.  NT: tiles of 8 tokens.
template <typename T, typename TG, bool NORM, bool FUSED, int NT>
__global__ void __launch_bounds__(THREADS, 1) stream_kernel(const Int8ProductParams P, const Int8RowsParams R, const Plan plan, int mode, int out_f32) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float token_scale[NT * 8], sums[WARPS];
  __shared__ uint32_t tops[WARPS];
  unsigned char* ring = smem;
  int* red = reinterpret_cast<int*>(smem + RING);                               // [2][WARPS][NT * 8 tokens][16 rows]
  int8_t* xs = reinterpret_cast<int8_t*>(red + 2 * WARPS * NT * 128);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int wn = warp / plan.wk, wk = warp % plan.wk;
  const bool glu = mode == INT8_GLU;

  // this thread's two weight rows of a unit
  const int8_t *p0, *p1;
  bool v0, v1;
  auto rows_of = [&](int unit) {
    const int r0 = unit * (glu ? 8 : 16) + g, r1 = glu ? r0 : r0 + 8;
    v0 = r0 < P.n;
    v1 = r1 < P.n;
    p0 = P.w + static_cast<size_t>(v0 ? r0 : 0) * P.w_pitch + t * 16;
    p1 = P.w + static_cast<size_t>((glu ? P.n : 0) + (v1 ? r1 : 0)) * P.w_pitch + t * 16;
  };
  const int first = blockIdx.x + gridDim.x * wn, stride = gridDim.x * plan.wn;
  int unit_in = first, step_in = 0;                                             // what is copied next
  rows_of(unit_in < plan.units ? unit_in : 0);
  for (int d = 0; d < DEPTH && d < plan.steps && first < plan.units; ++d) {
    const int at = (wk + d * plan.wk) * 64;
    if (at + t * 16 < P.k) {
      if (v0) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(p0 + at));
      if (v1) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(p1 + at));
    }
  }
  pdl_launch_dependents();
  pdl_wait();

  auto copy = [&](int slot) {
    if (unit_in < plan.units) {
      const int at = (wk + step_in * plan.wk) * 64;
      const bool in = at + t * 16 < P.k;
      unsigned char* dst = ring + (slot * 2 * THREADS + threadIdx.x) * 16;
      cp_async16(dst, in ? p0 + at : p0, in && v0);
      cp_async16(dst + THREADS * 16, in ? p1 + at : p1, in && v1);
      if (++step_in == plan.steps) {
        step_in = 0;
        unit_in += stride;
        if (unit_in < plan.units) rows_of(unit_in);
      }
    }
    cp_async_commit();
  };
  if constexpr (!FUSED) {
    const int pieces = plan.x_pitch / 16;
    for (int i = threadIdx.x; i < P.tokens * pieces; i += THREADS) {
      const int row = i / pieces, at = (i - row * pieces) * 16, left = P.k - at;         // (what lies beyond the row reads as 0)
      const int8_t* from = P.q + row * P.q_pitch + (left > 0 ? at : 0);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(xs + row * plan.x_pitch + at)), "l"(from), "r"(max(0, min(16, left))));
    }
    cp_async_commit();
  }
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) copy(d);

  if constexpr (FUSED) {
    tokens_to_8_bits<T, TG, NORM>(R, xs, plan.x_pitch, token_scale, sums, tops);
  } else {
    if (threadIdx.x < P.tokens) token_scale[threadIdx.x] = P.s[threadIdx.x];
    cp_async_wait<DEPTH>();                                                     // (the tokens; the weights behind them are on their way)
  }
  __syncthreads();

  // The scales (and bias) of the result that this thread finishes first come while the unit's products run.
  const int rows = glu ? 8 : 16, mine_first = wk * 32 + lane, mine_row = mine_first & (rows - 1);
  int slot = 0, turn = 0;
  for (int unit = first; unit < plan.units; unit += stride, turn ^= 1) {
    int acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0;
    const int col = unit * rows + mine_row;
    float c0 = 0.0f, c1 = 0.0f, b0 = 0.0f, b1 = 0.0f;
    if (mine_first < P.tokens * rows && col < P.n) {
      c0 = P.c[col];
      if (glu) c1 = P.c[P.n + col];
      if (P.bias) {
        b0 = P.bias[col];
        if (glu) b1 = P.bias[P.n + col];
      }
    }
    for (int i = 0; i < plan.steps; ++i) {
      const int at = (wk + i * plan.wk) * 64 + t * 16;
      uint4 x[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j)
        x[j] = at < P.k && j * 8 + g < P.tokens ? *reinterpret_cast<const uint4*>(xs + (j * 8 + g) * plan.x_pitch + at) : make_uint4(0u, 0u, 0u, 0u);
      cp_async_wait<DEPTH - 1>();
      const unsigned char* src = ring + (slot * 2 * THREADS + threadIdx.x) * 16;
      const uint4 a = own_piece(src), b = own_piece(src + THREADS * 16);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        mma_s8(acc[j], a.x, b.x, a.y, b.y, x[j].x, x[j].y);
        mma_s8(acc[j], a.z, b.z, a.w, b.w, x[j].z, x[j].w);
      }
      copy(slot);
      slot = slot + 1 == DEPTH ? 0 : slot + 1;
    }
    int* mine = red + (turn * WARPS + warp) * NT * 128;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[(j * 8 + t * 2 + (e & 1)) * 16 + g + (e >> 1) * 8] = acc[j][e];
    asm volatile("bar.sync %0, %1;\n" ::"r"(1 + wn), "r"(plan.wk * 32) : "memory");       // the group's warps
    // (a thread's further results are of other tokens, in the same column: their number is a multiple of the rows)
    for (int i = mine_first; i < P.tokens * rows; i += plan.wk * 32) {
      if (col >= P.n) continue;
      const int token = glu ? i >> 3 : i >> 4;
      const int* from = red + (turn * WARPS + wn * plan.wk) * NT * 128 + token * 16 + mine_row;
      int sum = 0, up = 0;
      for (int w = 0; w < plan.wk; ++w) {
        sum += from[w * NT * 128];
        if (glu) up += from[w * NT * 128 + 8];
      }
      float z = fmaf(static_cast<float>(sum), token_scale[token] * c0, b0);
      if (glu) {
        const float u = fmaf(static_cast<float>(up), token_scale[token] * c1, b1);
        z = out_f32 ? gate_up<true>(z, u, P.limit, P.alpha) : gate_up<false>(z, u, P.limit, P.alpha);
      }
      const size_t at = static_cast<size_t>(token) * P.n + col;
      if (out_f32) static_cast<float*>(P.out)[at] = z;
      else static_cast<__nv_bfloat16*>(P.out)[at] = __float2bfloat16_rn(z);
    }
  }
}

// ------------------------------------------------------------------ host side
static inline int x_pitch_of(int k) {                            // an odd number of 64-byte pieces: tokens meet in no bank
  const int p = (k + 63) / 64;
  return (p | 1) * 64;
}
static inline int smem_of(int tokens, int k) {
  return RING + 2 * WARPS * (tokens > 8 ? 2 : 1) * 512 + tokens * x_pitch_of(k);
}
// Whether a thread can hold its share of the tokens' floats, with one kernel for everything.
static inline bool fuses(int tokens, int k) {
  const int slots = tokens <= 1 ? 1 : tokens <= 2 ? 2 : tokens <= 4 ? 4 : 8;
  return tokens <= 8 && (k + 7) / 8 <= INT8_ROW_CHUNKS * THREADS / slots;
}
static inline bool takes(int tokens, int k) { return tokens <= MOST_TOKENS && smem_of(tokens, k) <= DYNAMIC_MOST; }

static inline Plan make_plan(int n, int k, int mode, int sms) {
  Plan p;
  const int steps = (k + 63) / 64, rows = mode == INT8_GLU ? 8 : 16;
  p.units = (n + rows - 1) / rows;
  long long best = 0;
  for (int wn = 1; wn <= 4; wn *= 2) {
    const int wk = WARPS / wn, share = (steps + wk - 1) / wk;
    // Rounds of the fullest group, each its steps and about four more for the sums' meeting and a late group's wait; from sixteen
    // units an SM on rounds even out, and a unit that all warps share is the fastest.  (One token, WN = 1, 2, 4, us: 24,576 x 4,096
    // gated 19.3, 18.9, 18.1; 6,144 x 4,096 7.2, 6.9, 6.3; 4,096 x 12,288 11.2, 10.7, 11.4; 4,096 x 1,024 3.7, 2.8, 2.8; 151,936 x 4,096
    // 92.0, 94.1, 94.7.)
    if (wn > 1 && p.units >= 16 * sms) break;
    const long long groups = static_cast<long long>(sms) * wn, cost = (p.units + groups - 1) / groups * (share + 4);
    if (best == 0 || cost < best) {
      best = cost;
      p.wn = wn; p.wk = wk; p.steps = share;
    }
  }
  p.x_pitch = x_pitch_of(k);
  return p;
}

template <typename T, typename TG, bool NORM, bool FUSED, int NT>
static int launch_one(const Int8ProductParams& P, const Int8RowsParams& R, int mode, int out_code, const Int8Device& device, cudaStream_t stream) {
  static bool set[64];
  const int rc = int8_launch_limit(stream_kernel<T, TG, NORM, FUSED, NT>, DYNAMIC_MOST, device, set);
  if (rc != 0) return rc;
  const Plan plan = make_plan(P.n, P.k, mode, device.sms);
  return b200_launch(stream_kernel<T, TG, NORM, FUSED, NT>, dim3(plan.units < device.sms ? plan.units : device.sms), dim3(THREADS), smem_of(P.tokens, P.k), stream,
                     0, P, R, plan, mode, static_cast<int>(out_code == B200_F32));
}

// `R`: the tokens as floats (null: P.q and P.s are there already).
static int product(const Int8ProductParams& P, const Int8RowsParams* R, int x_code, int gain_code, int mode, int out_code, const Int8Device& device, cudaStream_t stream) {
  const Int8RowsParams none = {};
  if (R == nullptr)
    return P.tokens > 8 ? launch_one<float, float, false, false, 2>(P, none, mode, out_code, device, stream)
                        : launch_one<float, float, false, false, 1>(P, none, mode, out_code, device, stream);
  const bool wide_x = x_code == B200_F32, wide_g = gain_code == B200_F32;
  if (R->gain == nullptr)
    return wide_x ? launch_one<float, float, false, true, 1>(P, *R, mode, out_code, device, stream)
                  : launch_one<__nv_bfloat16, float, false, true, 1>(P, *R, mode, out_code, device, stream);
  if (wide_x)
    return wide_g ? launch_one<float, float, true, true, 1>(P, *R, mode, out_code, device, stream)
                  : launch_one<float, __nv_bfloat16, true, true, 1>(P, *R, mode, out_code, device, stream);
  return wide_g ? launch_one<__nv_bfloat16, float, true, true, 1>(P, *R, mode, out_code, device, stream)
                : launch_one<__nv_bfloat16, __nv_bfloat16, true, true, 1>(P, *R, mode, out_code, device, stream);
}

}  // namespace i8st
