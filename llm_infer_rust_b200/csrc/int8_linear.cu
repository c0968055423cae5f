// Products in 8-bit integers: out[t, n] = s[t] c[n] sum_k q[t, k] w[n, k] (+ bias[n]), or behind packed gate and up rows
// act(gate) * up of those floats.  q, s: the tokens in 8 bits (int8_rows.cuh), w, c: the weights, one scale a row.
//
// The sums are 32-bit integers and exact: |q|, |w| <= 128 and K <= 131,071 keep them below 2^31, so their order does not
// matter.  The scales are multiplied in float and the result is rounded once, to the output's type.
#include <math.h>

#include "int8_rows.cuh"
#include "int8_stream.cuh"
#include "int8_tcgen05.cuh"

constexpr int MAX_K = 131071;
// Tokens and weight rows of a call.  Kernels count them in 32-bit integers and step past the end by what a grid takes at once: up to
// 9,472 rows to 8 bits, a tile of 256.
constexpr int MAX_ROWS = 2147483647 - 65536;

static Int8Device current_device() {
  static int counts[64];                       // SMs of the devices that were asked (0: not yet)
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return {-1, 148};
  if (device >= 64) return {device, 148};
  if (counts[device] == 0) cudaDeviceGetAttribute(&counts[device], cudaDevAttrMultiProcessorCount, device);
  return {device, counts[device] > 0 ? counts[device] : 148};
}

static int tiled_product(const Int8ProductParams& P, int mode, int out_code, const Int8Device& device, cudaStream_t stream) {
  if (mode == INT8_GLU)
    return out_code == B200_F32 ? i8tc::product<float, INT8_GLU>(P, device, stream) : i8tc::product<__nv_bfloat16, INT8_GLU>(P, device, stream);
  return out_code == B200_F32 ? i8tc::product<float, INT8_PLAIN>(P, device, stream) : i8tc::product<__nv_bfloat16, INT8_PLAIN>(P, device, stream);
}

// ------------------------------------------------------------------ entry points
static int rows_params(Int8RowsParams& R, const void* x, const void* residual, const void* gain, void* sum_out, void* q, float* s,
                       int tokens, int k, long long x_pitch, long long q_pitch, int x_code, int gain_code, float eps) {
  if ((x_code != B200_F32 && x_code != B200_BF16) || (gain && gain_code != B200_F32 && gain_code != B200_BF16)) return B200_BAD_DTYPE;
  if (tokens < 0 || tokens > MAX_ROWS || k < 1 || k > MAX_K || x_pitch < k || q_pitch < k) return B200_BAD_SIZE;
  if (!int8_aligned(q, q_pitch)) return B200_BAD_ALIGN;
  const long long e = x_code == B200_F32 ? 4 : 2;
  const bool whole = k % 8 == 0 && int8_aligned(x, x_pitch * e) && int8_aligned(residual, residual ? k * e : 0) && int8_aligned(gain, 0) &&
                    int8_aligned(sum_out, sum_out ? k * e : 0);
  R = {x, residual, gain, sum_out, static_cast<int8_t*>(q), s, tokens, k, x_pitch, q_pitch, eps, whole};
  return 0;
}

// q, s of `tokens` rows of x; gain null: no norm.
B200_EXPORT int b200_int8_rows(const void* x, const void* residual, const void* gain, void* sum_out, void* q, float* s, int tokens,
                               int k, long long x_pitch, long long q_pitch, int x_code, int gain_code, float eps, cudaStream_t stream) {
  Int8RowsParams R;
  const int rc = rows_params(R, x, residual, gain, sum_out, q, s, tokens, k, x_pitch, q_pitch, x_code, gain_code, eps);
  if (rc != 0 || tokens == 0) return rc;
  return !x || !q || !s ? B200_BAD_SIZE : int8_rows_launch(R, x_code, gain_code, current_device().sms, stream);
}

// 1 where the product of `tokens` rows of floats takes them to 8 bits itself: no place for q and s is needed.
B200_EXPORT int b200_int8_alone(int tokens, int k) {
  return k >= 1 && k <= MAX_K && i8st::takes(tokens, k) && i8st::fuses(tokens, k) ? 1 : 0;
}

// The shared memory that the streaming kernel asks for at launch with `tokens` rows of k columns (0: the tiled kernel takes them), and the
// most that it may ask for.
B200_EXPORT int b200_int8_stream_bytes(int tokens, int k) {
  return tokens >= 1 && k >= 1 && k <= MAX_K && i8st::takes(tokens, k) ? i8st::smem_of(tokens, k) : 0;
}
B200_EXPORT int b200_int8_stream_limit() { return i8st::DYNAMIC_MOST; }

// How the tiled product is cut up: 1,000 times the way (0: pairs of CTAs, else the CTAs that share a tile's k) plus the columns.
B200_EXPORT int b200_int8_plan(int tokens, int n, int k, int mode, int sms, int quads) {
  const i8tc::Plan p = i8tc::make_plan(tokens, n, k, mode, sms, quads, i8tc::smem_fixed<__nv_bfloat16>());
  return 1000 * p.way + p.bn;
}

// The product; `x` not null: of its rows, which go to q, s first (null where
// b200_int8_alone says so).
B200_EXPORT int b200_int8_linear(const void* x, const void* residual, const void* gain, void* sum_out, void* q, float* s,
                                 const void* w, const float* c, const float* bias, void* out, int tokens, int n, int k,
                                 long long x_pitch, long long q_pitch, long long w_pitch, int x_code, int gain_code, int out_code,
                                 int mode, float eps, float limit, float alpha, int* err, cudaStream_t stream) {
  if (out_code != B200_F32 && out_code != B200_BF16) return B200_BAD_DTYPE;
  if (tokens < 0 || tokens > MAX_ROWS || n < 0 || n > MAX_ROWS / (mode == INT8_GLU ? 2 : 1) || k < 1 || k > MAX_K || q_pitch < k || w_pitch < k ||
      (mode != INT8_PLAIN && mode != INT8_GLU))
    return B200_BAD_SIZE;
  if (!int8_aligned(q, q_pitch) || !int8_aligned(w, w_pitch)) return B200_BAD_ALIGN;
  if (tokens == 0) return 0;
  if ((!x && (!q || !s)) || (n > 0 && (!w || !c || !out))) return B200_BAD_SIZE;
  const Int8Device device = current_device();
  const bool few = n > 0 && i8st::takes(tokens, k);
  const Int8ProductParams P = {static_cast<const int8_t*>(q), s, static_cast<const int8_t*>(w), c, bias, out, tokens, n, k,
                               q_pitch, w_pitch, limit, alpha, err};
  const bool no_word = n > 0 && !err;           // (where a wait that runs out is flagged)
  if (x) {
    Int8RowsParams R;
    int rc = rows_params(R, x, residual, gain, sum_out, q, s, tokens, k, x_pitch, q_pitch, x_code, gain_code, eps);
    if (rc == 0 && no_word) rc = B200_BAD_SIZE;
    if (rc == 0 && few && i8st::fuses(tokens, k)) return i8st::product(P, &R, x_code, gain_code, mode, out_code, device, stream);
    if (rc == 0 && (q == nullptr || s == nullptr)) rc = B200_BAD_SIZE;
    if (rc == 0) rc = int8_rows_launch(R, x_code, gain_code, device.sms, stream);
    if (rc != 0) return rc;
  }
  if (n == 0) return 0;
  if (no_word) return B200_BAD_SIZE;
  return few ? i8st::product(P, nullptr, 0, 0, mode, out_code, device, stream) : tiled_product(P, mode, out_code, device, stream);
}
