// Shapes, the workspace layout and the split-KV schedule shared by the decode, schedule and combine kernels.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace mla {

constexpr int CKV = 512;          // latent channels (packed E2M1, 256 bytes per token)
constexpr int KPE = 64;           // rope channels (E4M3)
constexpr int TOKEN_BYTES = 352;  // 256 + 32 + 64
constexpr int TILE = 128;         // tokens per tile = rows of one tcgen05 MMA
constexpr int HALF = 64;          // tokens per staging slot

// One unit of work of a decode CTA: `ntiles` consecutive 128-token tiles of request `b`, head group `hg`, starting
// at token `tok0`; tokens at or beyond `tok_end` are masked. Its partial result goes to slot `cta + w`.
struct Seg {
  int b, hg, tok0, ntiles, tok_end, w, cta, pad;
};
static_assert(sizeof(Seg) == 32, "Seg is read as two 16-byte words");

// Workspace (device memory owned by the caller):
//   header     16 x int32   [0] error status (sticky), [1] total tiles, [2] tiles per CTA
//   cta_range  n_cta x int2 items [first, last) that intersect the CTA's tile range
//   item_range W x int2     CTAs [first, last] that hold a piece of item w (last < first: the item is empty)
//   segs       (n_cta + W) x Seg, indexed by slot = cta + w
//   lse_part   (n_cta + W) x heads_per_cta floats, log2 units
//   o_part     (n_cta + W) x heads_per_cta x 512 floats, each normalised by its own sum
struct WsLayout {
  size_t header, cta_range, item_range, segs, lse_part, o_part, total;
};
__host__ __device__ inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }
__host__ __device__ inline WsLayout ws_layout(int n_cta, long long W, int heads_per_cta) {
  WsLayout l;
  const size_t slots = size_t(n_cta) + size_t(W);
  size_t off = 0;
  l.header = off, off = align_up(off + 64, 256);
  l.cta_range = off, off = align_up(off + size_t(n_cta) * 8, 256);
  l.item_range = off, off = align_up(off + size_t(W) * 8, 256);
  l.segs = off, off = align_up(off + slots * sizeof(Seg), 256);
  l.lse_part = off, off = align_up(off + slots * heads_per_cta * 4, 256);
  l.o_part = off, off = align_up(off + slots * heads_per_cta * CKV * 4, 256);
  l.total = off;
  return l;
}

// Item numbering: w = (b * splits + z) * head_groups + hg, so that the head groups of one (request, split) are
// neighbours in the flattened tile order and re-read the same KV range close together in time.
enum Map { kMapNone, kMapWindow, kMapChunk };  // how a batch entry's tokens are found: all of its request, or by a WindowMap
struct Problem {
  int batch, heads, heads_per_cta, head_groups, splits, chunk, n_cta;
  // Windowed decode and query tokens of chunks (splits 1), see WindowMap. window 0: none. pt_width: columns of the page table.
  // kMapChunk: batch entry b is query token q_first + b of the `requests` requests whose tokens q_indptr delimits
  int window, sinks, page_shift, pt_width, requests, q_first;
  const int* q_indptr;
  __host__ __device__ long long items() const { return (long long)batch * splits * head_groups; }
};

// the request whose rows [indptr[b], indptr[b + 1]) hold row i (indptr[0] <= i < indptr[batch]); empty requests hold none
__device__ __forceinline__ int request_of_row(const int* __restrict__ indptr, int batch, int i) {
  int lo = 0, hi = batch - 1;  // last b with indptr[b] <= i
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(indptr + mid) <= i) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Sliding-window decode. The query token of a request of n tokens sees the first S tokens and the last W: [0, S) and [n - W, n).
// Attention does not care about the numbering of the tokens, so the kernels get a shorter request instead of a second range: the
// first tokens' pages followed by the window's, the number of tokens up to the end of that, and the one interval of it that is not
// seen (what is left of the last of the first tokens' pages, and of the window's first page before the window begins). Everything
// that schedules, loads and multiplies then works on visible pages alone; the kernels mask the interval. A query token of a chunk is
// treated like a request that ends with it; one of no request sees nothing.
struct WindowMap {
  int request;         // row of the page table
  int len;             // tokens of the shortened request
  int first, skipped;  // pages: the first tokens' ones, and how many follow them that are left out
  int2 dead;           // tokens of the shortened request that are not seen
  __device__ __forceinline__ int page(int i) const { return i < first ? i : i + skipped; }  // of the request, for page i of the shortened one
};
__device__ __forceinline__ WindowMap window_map(int request, int n, int window, int sinks, int page_shift) {
  const int begin = window > 0 && n > window ? n - window : 0;  // first token of the window
  const int bp = begin >> page_shift;
  WindowMap m;
  m.request = request;
  m.first = int(min((long long)bp, ((long long)sinks + (1ll << page_shift) - 1) >> page_shift));
  m.skipped = bp - m.first;
  m.len = n - (m.skipped << page_shift);
  m.dead = make_int2(sinks, max(sinks, begin - (m.skipped << page_shift)));
  return m;
}
template <int MAP>
__device__ __forceinline__ WindowMap window_map(const int* kv_lens, const Problem& pb, int b) {
  const long long most = (long long)pb.pt_width << pb.page_shift;  // a length past the page table is cut at its end
  int request = b, behind = 0;  // tokens behind the query token
  if constexpr (MAP == kMapChunk) {
    const int at = pb.q_first + b;
    if (at < pb.q_indptr[0] || at >= pb.q_indptr[pb.requests]) return window_map(0, 0, pb.window, pb.sinks, pb.page_shift);
    request = request_of_row(pb.q_indptr, pb.requests, at);
    behind = pb.q_indptr[request + 1] - 1 - at;
  }
  const int n = kv_lens[request];
  return window_map(request, (n < most ? n : int(most)) - behind, pb.window, pb.sinks, pb.page_shift);
}
// tokens of request b that are scheduled
template <int MAP>
__device__ __forceinline__ int sched_len(const int* kv_lens, const Problem& pb, int b) {
  if constexpr (MAP != kMapNone) return window_map<MAP>(kv_lens, pb, b).len;
  else return kv_lens[b];
}

// 128-token tiles of (request, split) pair bz = b * splits + z: the split covers tokens [z * chunk, (z + 1) * chunk) of the request.
__device__ __forceinline__ int sched_tiles(int len, const Problem& pb, int bz) {
  long long n = (long long)len - (long long)(bz % pb.splits) * pb.chunk;
  n = n < 0 ? 0 : (n > pb.chunk ? pb.chunk : n);
  return int((n + TILE - 1) / TILE);
}

enum Status : int {
  kOk = 0,
  kWaitTimeout = 1,   // a bounded wait inside the decode kernel gave up
  kBadSchedule = 2,   // schedule kernel: batch * splits exceeds its scan capacity
  kBadPage = 3,       // a page id of a request's live range lies outside [0, num_pages): its rows were not loaded
  kPeerTimeout = 4,   // cross-GPU merge: another GPU's record was not announced within the wait limit
};

}  // namespace mla
