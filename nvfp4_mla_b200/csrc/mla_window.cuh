// A few query tokens per request through the decode kernels: every token becomes a request of its own, with the page table, the length
// and the unseen interval that its window leaves (WindowMap, mla_common.cuh).
#pragma once
#include "mla_common.cuh"
#include "mla_gather.cuh"  // request_of_row
#include "ptx_sm100.cuh"

namespace mla {

constexpr int kWindowThreads = 128;

// The query tokens of a chunk, each as a request of its own: token i belongs to the request b with indptr[b] <= i < indptr[b + 1] and
// sees the tokens up to its own position, kv_lens[b] - (indptr[b + 1] - i). A token of no request sees nothing.
struct ChunkTokens {
  const int* indptr;
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
  const int at = chunk.first + i;
  int b = -1, n = 0;
  if (at >= chunk.indptr[0] && at < chunk.indptr[chunk.batch]) {
    b = request_of_row(chunk.indptr, chunk.batch, at);
    n = kv_lens[b] - (chunk.indptr[b + 1] - 1 - at);
  }
  const WindowMap m = window_map(n, window, sinks, page_shift);
  int pages = int(((long long)(m.len > 0 ? m.len : 0) + (1 << page_shift) - 1) >> page_shift);
  pages = pages < width ? pages : width;
  for (int k = lane; k < pages; k += 32) {
    const int page = m.page(k);
    table[(long long)i * width + k] = page < pt_width ? page_table[(long long)b * pt_stride + page] : -1;
  }
  if (lane == 0) {
    const long long most = (long long)width << page_shift;
    lens[i] = m.len < most ? m.len : int(most);
    dead[i] = m.dead;
  }
}

}  // namespace mla
