// Copies of cache pages, in the tensors of all layers in one launch.
//
// A move (source, target, n) makes slots 0 .. n - 1 of page `target` those of page `source`, in every tensor
// [pages, heads, page_size, dim] of a table: heads runs of n * dim elements, n * dim * page_size apart.  The moves are checked
// on the host (pages in range, no page written twice, none both read and written), so they may run in any order, and reach
// the kernel as its parameters: a call needs no upload and nothing of the caller's has to outlive it.
//
// The bytes bound it, and where they are few the launch.  A CTA takes a piece of one page of one tensor; a thread has four
// vectors on their way.  A source with several targets is read from memory once and from the second-level cache behind that.
#include <stdlib.h>
#include <string.h>

#include "common.cuh"

struct PageTensor {                        // 32 bytes, in device memory, made once with the cache
  unsigned char* base;
  long long page_bytes;                    // heads * page_size * row
  int head_bytes;                          // page_size * row
  int row;                                 // bytes of a token of one head
  int heads, pad;
};
struct PageMove { int source, target, slots; };
template <int MOST>
struct PageMoves { PageMove move[MOST]; };

constexpr int THREADS = 256, UNROLL = 4;
constexpr int FEW_MOVES = 64, MOST_MOVES = 2048;      // of a launch: 768 bytes or 24 KB of parameters (more moves take more launches)

// grid (tensors * pieces, moves).  V: what all addresses and rows are multiples of.
template <typename V, int MOST>
__global__ void __launch_bounds__(THREADS)
copy_pages_kernel(const __grid_constant__ PageMoves<MOST> moves, const PageTensor* __restrict__ tensors, int pieces, int page_size) {
  const PageTensor t = tensors[blockIdx.x / pieces];
  const PageMove m = moves.move[blockIdx.y];
  if (m.slots == 0) return;
  // runs of `length` vectors, `apart` from one to the next; a whole page is one run
  const bool whole = m.slots == page_size;
  const int runs = whole ? 1 : t.heads;
  const int length = (whole ? static_cast<int>(t.page_bytes / sizeof(V)) : m.slots * (t.row / static_cast<int>(sizeof(V))));
  const int apart = t.head_bytes / static_cast<int>(sizeof(V));
  const V* from = reinterpret_cast<const V*>(t.base + m.source * t.page_bytes);
  V* to = reinterpret_cast<V*>(t.base + m.target * t.page_bytes);
  const int step = pieces * THREADS, step_runs = step / length, step_rest = step - step_runs * length;
  int run = (static_cast<int>(blockIdx.x) % pieces * THREADS + static_cast<int>(threadIdx.x)) / length;
  int off = (static_cast<int>(blockIdx.x) % pieces * THREADS + static_cast<int>(threadIdx.x)) - run * length;
  while (run < runs) {
    V v[UNROLL];
    int at[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      at[u] = run < runs ? run * apart + off : -1;
      if (at[u] >= 0) v[u] = from[at[u]];
      run += step_runs;
      off += step_rest;
      if (off >= length) { off -= length; ++run; }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (at[u] >= 0) to[at[u]] = v[u];
  }
}

enum : int { PAGES_OUTSIDE = -10, PAGES_TWICE = -11, PAGES_NO_MEMORY = -12 };

// What the moves must be: pages 0 .. pages - 1, 0 to page_size slots, no target twice and none that is a source.
static int check_moves(const PageMove* moves, int n, long long pages, int page_size) {
  for (int i = 0; i < n; ++i)
    if (moves[i].source < 0 || moves[i].source >= pages || moves[i].target < 0 || moves[i].target >= pages || moves[i].slots < 0 ||
        moves[i].slots > page_size)
      return PAGES_OUTSIDE;
  if (n <= 16) {                            // (a fork or two: compared pair by pair)
    for (int i = 0; i < n; ++i)
      for (int j = 0; j < n; ++j)
        if (moves[i].target == moves[j].source || (i != j && moves[i].target == moves[j].target)) return PAGES_TWICE;
    return 0;
  }
  unsigned char* written = static_cast<unsigned char*>(calloc(static_cast<size_t>(pages + 7) / 8, 1));
  if (written == nullptr) return PAGES_NO_MEMORY;
  int rc = 0;
  for (int i = 0; i < n && rc == 0; ++i) {
    unsigned char& byte = written[moves[i].target / 8];
    const unsigned char bit = static_cast<unsigned char>(1u << (moves[i].target % 8));
    if (byte & bit) rc = PAGES_TWICE;
    byte |= bit;
  }
  for (int i = 0; i < n && rc == 0; ++i)
    if (written[moves[i].source / 8] >> (moves[i].source % 8) & 1) rc = PAGES_TWICE;
  free(written);
  return rc;
}

template <typename V, int MOST>
static int launch(const PageMove* moves, int n, const PageTensor* tensors, int count, int pieces, int page_size, cudaStream_t stream) {
  PageMoves<MOST> some;
  memcpy(some.move, moves, sizeof(PageMove) * n);
  if (n < MOST) memset(some.move + n, 0, sizeof(PageMove) * (MOST - n));
  copy_pages_kernel<V, MOST><<<dim3(static_cast<unsigned>(count) * pieces, n), THREADS, 0, stream>>>(some, tensors, pieces, page_size);
  return b200_check_launch();
}
template <typename V>
static int launch_all(const PageMove* moves, int n, const PageTensor* tensors, int count, int pieces, int page_size, cudaStream_t stream) {
  for (int at = 0; at < n; at += MOST_MOVES) {
    const int some = n - at < MOST_MOVES ? n - at : MOST_MOVES;
    const int rc = some <= FEW_MOVES ? launch<V, FEW_MOVES>(moves + at, some, tensors, count, pieces, page_size, stream)
                                     : launch<V, MOST_MOVES>(moves + at, some, tensors, count, pieces, page_size, stream);
    if (rc != 0) return rc;
  }
  return 0;
}

// `moves`: host memory, n times (source, target, slots); `tensors`: device memory, `count` PageTensors of `pages` pages each;
// `vector`: 16, 4 or 2, which divides every base, row and page; `page_bytes`: of the largest page.  Moves of no slots do nothing.
B200_EXPORT int b200_copy_pages(const void* moves, int n, const void* tensors, int count, long long pages, int page_size, int vector,
                                long long page_bytes, cudaStream_t stream) {
  if (n == 0 || count == 0) return 0;
  if (n < 0 || count < 0 || pages <= 0 || page_size <= 0 || page_bytes <= 0 || moves == nullptr || tensors == nullptr) return B200_BAD_SIZE;
  if (page_bytes > (1 << 30)) return B200_BAD_SIZE;                   // (a page's vectors are counted in 32 bits)
  const PageMove* m = static_cast<const PageMove*>(moves);
  int rc = check_moves(m, n, pages, page_size);
  if (rc != 0) return rc;
  // Pieces of a page: enough CTAs for all SMs where there are few moves, no piece of less than a vector a thread.
  const long long most = (page_bytes / vector + THREADS - 1) / THREADS;
  long long pieces = (4 * 148 + static_cast<long long>(n) * count - 1) / (static_cast<long long>(n) * count);
  if (pieces > most) pieces = most;
  if (pieces * count > INT32_MAX) return B200_BAD_SIZE;
  const PageTensor* t = static_cast<const PageTensor*>(tensors);
  switch (vector) {
    case 16: return launch_all<uint4>(m, n, t, count, static_cast<int>(pieces), page_size, stream);
    case 4: return launch_all<uint32_t>(m, n, t, count, static_cast<int>(pieces), page_size, stream);
    case 2: return launch_all<uint16_t>(m, n, t, count, static_cast<int>(pieces), page_size, stream);
    default: return B200_BAD_ALIGN;
  }
}
