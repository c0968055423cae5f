// Products in 8-bit integers: out[t, n] = s[t] c[n] sum_k q[t, k] w[n, k] (+ bias[n]), or behind packed gate and up rows
// act(gate) * up of those floats.  q, s: the tokens in 8 bits (int8_rows.cuh), w, c: the weights, one scale a row.
//
// The sums are 32-bit integers and exact: |q|, |w| <= 128 and K <= 131,071 keep them below 2^31, so their order does not
// matter.  The scales are multiplied in float and the result is rounded once, to the output's type.
#include <math.h>

#include "int8_rows.cuh"

constexpr int MAX_K = 131071;

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
};

// 64 tokens x 64 columns a block, four bytes of k an instruction.
constexpr int TILE = 64, KB = 64;
template <typename T, int MODE>
__global__ void __launch_bounds__(256) int8_product_kernel(const Int8ProductParams P) {
  __shared__ uint32_t qs[TILE][KB / 4 + 1], ws[(MODE == INT8_GLU ? 2 : 1) * TILE][KB / 4 + 1];
  constexpr int HALVES = MODE == INT8_GLU ? 2 : 1;
  const int t0 = blockIdx.y * TILE, n0 = blockIdx.x * TILE;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  int acc[HALVES][4][4] = {};
  pdl_launch_dependents();
  pdl_wait();
  for (int k0 = 0; k0 < P.k; k0 += KB) {
    for (int i = threadIdx.x; i < TILE * KB; i += 256) {
      const int r = i / KB, k = i % KB;
      reinterpret_cast<int8_t*>(qs[r])[k] = t0 + r < P.tokens && k0 + k < P.k ? P.q[static_cast<size_t>(t0 + r) * P.q_pitch + k0 + k] : 0;
      for (int h = 0; h < HALVES; ++h)
        reinterpret_cast<int8_t*>(ws[h * TILE + r])[k] =
            n0 + r < P.n && k0 + k < P.k ? P.w[static_cast<size_t>(h * P.n + n0 + r) * P.w_pitch + k0 + k] : 0;
    }
    __syncthreads();
    for (int k = 0; k < KB / 4; ++k)
      for (int h = 0; h < HALVES; ++h)
        for (int i = 0; i < 4; ++i)
          for (int j = 0; j < 4; ++j)
            acc[h][i][j] = __dp4a(static_cast<int>(qs[ty + 16 * i][k]), static_cast<int>(ws[h * TILE + tx + 16 * j][k]), acc[h][i][j]);
    __syncthreads();
  }
  T* out = static_cast<T*>(P.out);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int t = t0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (t >= P.tokens || n >= P.n) continue;
      float y[HALVES];
      for (int h = 0; h < HALVES; ++h) {
        y[h] = static_cast<float>(acc[h][i][j]) * (P.s[t] * P.c[h * P.n + n]);
        if (P.bias) y[h] += P.bias[h * P.n + n];
      }
      out[static_cast<size_t>(t) * P.n + n] = from_f32<T>(MODE == INT8_GLU ? glu_product(y[0], y[HALVES - 1], P.limit, P.alpha) : y[0]);
    }
}

static int int8_product(const Int8ProductParams& P, int mode, int out_code, cudaStream_t stream) {
  auto kernel = mode == INT8_GLU ? (out_code == B200_F32 ? int8_product_kernel<float, INT8_GLU> : int8_product_kernel<__nv_bfloat16, INT8_GLU>)
                                 : (out_code == B200_F32 ? int8_product_kernel<float, INT8_PLAIN> : int8_product_kernel<__nv_bfloat16, INT8_PLAIN>);
  return b200_launch(kernel, dim3((P.n + TILE - 1) / TILE, (P.tokens + TILE - 1) / TILE), dim3(256), 0, stream, 0, P);
}

// ------------------------------------------------------------------ entry points
static int rows_params(Int8RowsParams& R, const void* x, const void* residual, const void* gain, void* sum_out, void* q, float* s,
                       int tokens, int k, long long x_pitch, long long q_pitch, int x_code, int gain_code, float eps) {
  if ((x_code != B200_F32 && x_code != B200_BF16) || (gain && gain_code != B200_F32 && gain_code != B200_BF16)) return B200_BAD_DTYPE;
  if (tokens < 0 || k < 1 || k > MAX_K || x_pitch < k || q_pitch < k) return B200_BAD_SIZE;
  if (!int8_aligned(q, q_pitch)) return B200_BAD_ALIGN;
  const long long e = x_code == B200_F32 ? 4 : 2;
  const bool wide = int8_aligned(x, x_pitch * e) && int8_aligned(residual, residual ? k * e : 0) && int8_aligned(gain, 0) &&
                    int8_aligned(sum_out, sum_out ? k * e : 0);
  R = {x, residual, gain, sum_out, static_cast<int8_t*>(q), s, tokens, k, x_pitch, q_pitch, eps, wide};
  return 0;
}

// q, s of `tokens` rows of x; gain null: no norm.
B200_EXPORT int b200_int8_rows(const void* x, const void* residual, const void* gain, void* sum_out, void* q, float* s, int tokens,
                               int k, long long x_pitch, long long q_pitch, int x_code, int gain_code, float eps, cudaStream_t stream) {
  Int8RowsParams R;
  const int rc = rows_params(R, x, residual, gain, sum_out, q, s, tokens, k, x_pitch, q_pitch, x_code, gain_code, eps);
  return rc != 0 ? rc : tokens == 0 ? 0 : int8_rows_launch(R, x_code, gain_code, stream);
}

// The product; `x` not null: of its rows, which go to q, s first.
B200_EXPORT int b200_int8_linear(const void* x, const void* residual, const void* gain, void* sum_out, void* q, float* s,
                                 const void* w, const float* c, const float* bias, void* out, int tokens, int n, int k,
                                 long long x_pitch, long long q_pitch, long long w_pitch, int x_code, int gain_code, int out_code,
                                 int mode, float eps, float limit, float alpha, int* err, cudaStream_t stream) {
  if (out_code != B200_F32 && out_code != B200_BF16) return B200_BAD_DTYPE;
  if (tokens < 0 || n < 0 || k < 1 || k > MAX_K || q_pitch < k || w_pitch < k || (mode != INT8_PLAIN && mode != INT8_GLU)) return B200_BAD_SIZE;
  if (!int8_aligned(q, q_pitch) || !int8_aligned(w, w_pitch)) return B200_BAD_ALIGN;
  if (tokens == 0) return 0;
  if (x) {
    Int8RowsParams R;
    int rc = rows_params(R, x, residual, gain, sum_out, q, s, tokens, k, x_pitch, q_pitch, x_code, gain_code, eps);
    if (rc == 0) rc = int8_rows_launch(R, x_code, gain_code, stream);
    if (rc != 0) return rc;
  }
  if (n == 0) return 0;
  const Int8ProductParams P = {static_cast<const int8_t*>(q), s, static_cast<const int8_t*>(w), c, bias, out, tokens, n, k,
                               q_pitch, w_pitch, limit, alpha};
  return int8_product(P, mode, out_code, stream);
}
