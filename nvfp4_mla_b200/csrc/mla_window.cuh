// Sliding-window decode: which pages a request's visible tokens are on.
//
// The query token of a request of n tokens sees the first S tokens and the last W: [0, S) and [n - W, n). Attention does not care
// about the order or the numbering of the tokens, so the decode kernels get a shorter request instead of a second range: a page
// table of the first tokens' pages followed by the window's, the number of tokens up to the end of that, and the one interval of it
// that is not seen (what is left of the last of the first tokens' pages, and of the window's first page before the window begins).
// Everything that schedules, loads and multiplies then works on visible pages alone; the kernels mask the interval.
#pragma once
#include "mla_common.cuh"
#include "mla_gather.cuh"  // request_of_row
#include "ptx_sm100.cuh"

namespace mla {

constexpr int kWindowThreads = 128;

// The query tokens of a chunk, each as a request of its own: token i belongs to the request b with indptr[b] <= i < indptr[b + 1] and
// sees the tokens up to its own position, kv_lens[b] - (indptr[b + 1] - i). A token of no request sees nothing.
struct ChunkTokens {
  const int* indptr;  // null: one query token per request
  int batch, first;   // requests; index of the first query token
};

// One warp per query token: a few dozen page ids. window 0: no window, all tokens up to its position are seen.
__global__ void __launch_bounds__(kWindowThreads)
mla_window_plan_kernel(const int* __restrict__ page_table, long long pt_stride, int pt_width, const int* __restrict__ kv_lens,
                       ChunkTokens chunk, int tokens, int page_shift, int window, int sinks, int width, int* __restrict__ table,
                       int* __restrict__ lens, int2* __restrict__ dead) {
  ptx::grid_launch_dependents();  // (the decode kernel waits for this grid before it reads)
  const int i = int(blockIdx.x) * (kWindowThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= tokens) return;
  int b = i, n = 0;
  if (chunk.indptr) {
    const int at = chunk.first + i;
    b = -1;
    if (at >= chunk.indptr[0] && at < chunk.indptr[chunk.batch]) {
      b = request_of_row(chunk.indptr, chunk.batch, at);
      n = kv_lens[b] - (chunk.indptr[b + 1] - 1 - at);
    }
  } else {
    n = kv_lens[i];
  }
  const int begin = window > 0 && n > window ? n - window : 0;                        // first token of the window
  const int first = int(((long long)sinks + (1ll << page_shift) - 1) >> page_shift);  // pages of the first tokens
  const int skipped = (begin >> page_shift) > first ? (begin >> page_shift) - first : 0;  // pages between them and the window
  const int shift = skipped << page_shift;
  int pages = int(((long long)(n > 0 ? n : 0) - shift + (1 << page_shift) - 1) >> page_shift);
  pages = pages < width ? pages : width;
  for (int k = lane; k < pages; k += 32) {
    const int at = k < first ? k : k + skipped;
    table[(long long)i * width + k] = at < pt_width ? page_table[(long long)b * pt_stride + at] : -1;
  }
  if (lane == 0) {
    const long long most = (long long)width << page_shift;
    lens[i] = n - shift < most ? n - shift : int(most);
    dead[i] = begin > sinks ? make_int2(sinks, begin - shift) : make_int2(0, 0);
  }
}

}  // namespace mla
