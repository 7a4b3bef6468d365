// Chunks of new tokens, everything around the attention kernel (mla_extend_sm100.cuh): the schedule, the FP16 operands, the merge.
//
// The rows of a request (query token, head) are cut into tiles of 128, the ITEMS; an item's work is the 256-token tiles of the cache
// that its rows see. The items' tiles are laid end to end and cut into equal pieces, one per CTA pair.
//
// Window: the tokens that some query of the request sees are [0, S) and everything from the first query's window on. The cache is
// read into a numbering of tiles that has no gap: the first `sink_tiles` tiles, then the tiles from the window's on, `shift` tokens
// further in the request. An item skips the tiles between the first tokens' and its own window.
//
// Operands: the attention kernel multiplies FP16. Every visible token is dequantised once per call into a workspace row of 576 (latent
// 512, rope 64, exact: e2m1 x e4m3 has six significant bits), every query row once into a row of the same shape, held times a power
// of two that puts its maximum into [2^14, 2^15) (the latent part stays exact down to 2^-39 of the maximum) with the rope part times
// kpe_scale / ckv_scale, rounded to FP16. 1.5 KB per token, against 256 KB of operands that the attention loads per token and
// 128-row tile, if it is read by many tiles.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "mla_common.cuh"
#include "mla_gather.cuh"  // request_of_row
#include "mla_schedule.cuh"
#include "ptx_sm100.cuh"

namespace mla {

constexpr int kExtRows = 128;   // rows of an item
constexpr int kExtTile = 256;   // tokens of a tile
constexpr int kExtRow = CKV + KPE;
constexpr int kExtMaxBatch = 8192;

struct ExtItem {
  int prefix;      // tiles of the items before
  int ntiles;      // at least 1 (an item that sees nothing has one tile, all masked)
  int tile0;       // first workspace tile of the request
  int sinks, skip; // tiles: the first tokens' ones, and how many follow them that no row sees
  int shift;       // tokens: position of a token in the request minus its place in the request's workspace tiles, behind the first tokens' tiles
  int row0, rows;  // first row in [total_q * heads], number of rows
  int r0;          // first row within the request
  int pos0;        // position of the request's first query token
  int pad[6];
};
static_assert(sizeof(ExtItem) == 64, "ExtItem is a cache line half");

struct ExtPair {
  int item, first, count;  // first item, first flattened tile, tiles
  int split;               // item whose first tiles this pair holds and whose last ones another does, or -1
};

// What the caller gives and how much room there is
struct ExtProblem {
  const int* kv_lens;
  const int* indptr;
  int batch, total_q, heads, max_kv_len, window, sinks, pairs;
  int max_items, max_tiles;
  int* req_tile0;   // [batch + 1] workspace tiles before request b
  int* req_item0;   // [batch + 1] items before request b
  int4* req_map;    // [batch] {shift, first tokens' tiles, tokens in the tiles (with the shift taken out), first token of the window}
  ExtItem* items;   // [max_items]
  ExtPair* pair;    // [pairs]
  int* counts;      // [0] items, [1] workspace tiles
  int* status;
};

constexpr int kExtSchedThreads = 1024;

// inclusive scan over the block; `sums`: one int per warp
__device__ __forceinline__ int block_scan(int v, int* sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(~0u, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  int base = 0;
  for (int i = 0; i < warp; ++i) base += sums[i];
  return base + v;
}

struct ExtRequest {
  int q0, q, n, pos0, begin, shift, sink_tiles, tiles;
};
__device__ __forceinline__ ExtRequest ext_request(const ExtProblem& E, int b) {
  ExtRequest r;
  const int a = E.indptr[b], z = E.indptr[b + 1];
  const int lo = a < 0 ? 0 : a, hi = z < E.total_q ? z : E.total_q;
  r.q0 = lo, r.q = hi > lo ? hi - lo : 0;
  const int n = E.kv_lens[b];
  r.n = n < 0 ? 0 : n < E.max_kv_len ? n : E.max_kv_len;
  r.pos0 = r.n - (z - a) + (lo - a);
  r.shift = 0, r.sink_tiles = 0, r.begin = 0;
  if (E.window > 0) {
    const long long s = ((long long)E.sinks + kExtTile - 1) / kExtTile;
    const long long begin = (long long)r.pos0 - E.window + 1;  // first token in the window of the first query token
    r.begin = begin > 0 ? int(begin) : 0;
    const long long t = r.begin / kExtTile;
    if (t > s) r.shift = int(t - s) * kExtTile;
    r.sink_tiles = int(s < (r.n + kExtTile - 1) / kExtTile ? s : (r.n + kExtTile - 1) / kExtTile);
  }
  r.tiles = (r.n - r.shift + kExtTile - 1) / kExtTile;
  if (r.tiles < 1) r.tiles = 1;
  if (r.q == 0) r.tiles = 0;
  return r;
}

__global__ void __launch_bounds__(kExtSchedThreads, 1) mla_extend_schedule_kernel(const ExtProblem E) {
  __shared__ int item0[kExtMaxBatch + 1];
  __shared__ int sums[kExtSchedThreads / 32];
  ptx::grid_launch_dependents();
  const int tid = threadIdx.x;
  int items = 0, tiles = 0;
  for (int b0 = 0; b0 < E.batch; b0 += kExtSchedThreads) {
    const int b = b0 + tid;
    ExtRequest r = {};
    int mine = 0;
    if (b < E.batch) {
      r = ext_request(E, b);
      mine = int(((long long)r.q * E.heads + kExtRows - 1) / kExtRows);
    }
    const int ii = block_scan(mine, sums), it = block_scan(r.tiles, sums);
    if (b < E.batch) {
      item0[b] = items + ii - mine;
      E.req_item0[b] = items + ii - mine, E.req_tile0[b] = tiles + it - r.tiles;
      E.req_map[b] = make_int4(r.shift, r.sink_tiles, r.n - r.shift, r.begin);
    }
    __shared__ int last[2];
    if (tid == kExtSchedThreads - 1) last[0] = ii, last[1] = it;
    __syncthreads();
    items += last[0], tiles += last[1];
    __syncthreads();
  }
  // (a query index that runs backwards could ask for more than there is room for)
  if (items > E.max_items || tiles > E.max_tiles) {
    if (tid == 0 && E.status) atomicExch(E.status, int(kBadSchedule));
    items = 0, tiles = 0;
  }
  if (tid == 0) item0[E.batch] = items, E.req_item0[E.batch] = items, E.req_tile0[E.batch] = tiles, E.counts[0] = items, E.counts[1] = tiles;
  __syncthreads();
  int total = 0;
  for (int i0 = 0; i0 < items; i0 += kExtSchedThreads) {
    const int i = i0 + tid;
    ExtItem m = {};
    if (i < items) {
      int lo = 0, hi = E.batch - 1;  // last b with item0[b] <= i
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (item0[mid] <= i) lo = mid;
        else hi = mid - 1;
      }
      const ExtRequest r = ext_request(E, lo);
      m.r0 = (i - item0[lo]) * kExtRows;
      const long long rows = (long long)r.q * E.heads - m.r0;
      m.rows = int(rows < kExtRows ? rows : kExtRows);
      m.row0 = r.q0 * E.heads + m.r0, m.pos0 = r.pos0, m.shift = r.shift, m.tile0 = E.req_tile0[lo];
      const int first = r.pos0 + m.r0 / E.heads, last = r.pos0 + (m.r0 + m.rows - 1) / E.heads;  // positions of its query tokens
      const int end = last + 1 < r.n ? last + 1 : r.n;                                           // tokens before it are seen
      int e = (end - r.shift + kExtTile - 1) / kExtTile;                                         // tiles up to there
      m.sinks = 0, m.skip = 0;
      if (E.window > 0) {
        long long begin = (long long)first - E.window + 1 - r.shift;
        const int t = begin > 0 ? int(begin / kExtTile) : 0;
        m.sinks = r.sink_tiles;
        if (t > m.sinks) m.skip = t - m.sinks;
      }
      if (e > r.tiles) e = r.tiles;
      m.ntiles = e - m.skip;
      if (m.ntiles < 1) m.ntiles = 1, m.skip = 0;
    }
    const int incl = block_scan(m.ntiles, sums);
    if (i < items) {
      m.prefix = total + incl - m.ntiles;
      E.items[i] = m;
    }
    __shared__ int last_sum;
    if (tid == kExtSchedThreads - 1) last_sum = incl;
    __syncthreads();
    total += last_sum;
    __syncthreads();
  }
  const int q = total > 0 ? (total + E.pairs - 1) / E.pairs : 1;
  __threadfence_block();
  __syncthreads();
  for (int p = tid; p < E.pairs; p += kExtSchedThreads) {
    ExtPair o = {0, p * q, 0, -1};
    if ((long long)p * q < total) {
      o.count = total - o.first < q ? total - o.first : q;
      auto item_of = [&](int g) {
        int lo = 0, hi = items - 1;  // last item with prefix <= g
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (E.items[mid].prefix <= g) lo = mid;
          else hi = mid - 1;
        }
        return lo;
      };
      o.item = item_of(o.first);
      const int end = o.first + o.count, z = item_of(end - 1);
      if (E.items[z].prefix >= o.first && E.items[z].prefix + E.items[z].ntiles > end) o.split = z;
    }
    E.pair[p] = o;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Operands. Blocks [0, max_tiles): one 256-token tile of the workspace each; the others: one item's query rows each. All blocks
// share the rows of no request (zeros in the output).
// ---------------------------------------------------------------------------------------------------------------
struct ExtOperands {
  const __nv_bfloat16* q_nope;
  const __nv_bfloat16* q_pe;
  const uint8_t* ckv;
  const uint8_t* sf;
  const uint8_t* kpe;
  const int* page_table;
  long long pt_stride;
  int pt_width, page_shift, num_pages;
  float ckv_scale, kpe_scale, sm_scale_log2;
  __half* kv16;     // [max_tiles * 256][576]
  __half* q16;      // [max_items * 128][576]
  float* q_scale;   // [max_items * 128]: factor of a row's scores, log2 units
  uint4* out;       // [total_q * heads][512] BF16
};

constexpr int kExtPrepThreads = 256;

__device__ __forceinline__ void ext_convert_tile(const ExtProblem& E, const ExtOperands& O, int tile) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int lo = 0, hi = E.batch - 1;  // last b with req_tile0[b] <= tile
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (E.req_tile0[mid] <= tile) lo = mid;
    else hi = mid - 1;
  }
  const int4 map = E.req_map[lo];
  const int v = (tile - E.req_tile0[lo]) * kExtTile + 32 * warp + lane;  // this lane's token among the request's
  int src = -1;                                                          // its cache row; -1: zeros
  if (v < map.z) {
    const int tok = v < map.y * kExtTile ? v : v + map.x;
    // (tokens between the first ones and the window belong to tiles that are read, but their pages may be gone)
    if (tok < E.sinks || tok >= map.w) {
      const int pi = tok >> O.page_shift;
      const int page = pi < O.pt_width ? O.page_table[(long long)lo * O.pt_stride + pi] : -1;
      if (page >= 0 && page < O.num_pages) src = (page << O.page_shift) + (tok & ((1 << O.page_shift) - 1));
      else if (E.status) atomicExch(E.status, int(kBadPage));
    }
  }
  __half* const dst = O.kv16 + ((long long)tile * kExtTile + 32 * warp) * kExtRow;
  constexpr int U = 4;
#pragma unroll 1
  for (int i = 0; i < 32; i += U) {
    uint2 w[U];
    uint32_t sc[U], rp[U];
    int at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      at[u] = __shfl_sync(~0u, src, i + u);
      const long long row = at[u] < 0 ? 0 : at[u];
      w[u] = __ldg(reinterpret_cast<const uint2*>(O.ckv + row * (CKV / 2)) + lane);
      sc[u] = __ldg(O.sf + row * (CKV / 16) + lane);
      rp[u] = __ldg(reinterpret_cast<const uint16_t*>(O.kpe + row * KPE) + lane);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (at[u] < 0) sc[u] = 0, rp[u] = 0;
      // A NaN block scale must reach those rows alone that see the token, not those that multiply it with probability 0: the block
      // becomes 0 and the rope part, which only enters scores, NaN.
      const bool nan = (sc[u] & 0x7Fu) == 0x7Fu;
      const bool any = __any_sync(~0u, nan);
      if (nan) sc[u] = 0;
      const uint32_t s2 = ptx::e4m3x2_to_f16x2(uint16_t(sc[u] | sc[u] << 8));
      uint32_t a[4], b[4];
      ptx::e2m1x8_to_f16x8(w[u].x, a), ptx::e2m1x8_to_f16x8(w[u].y, b);
      uint4* const p = reinterpret_cast<uint4*>(dst + (long long)(i + u) * kExtRow) + 2 * lane;
      p[0] = make_uint4(ptx::hmul2(a[0], s2), ptx::hmul2(a[1], s2), ptx::hmul2(a[2], s2), ptx::hmul2(a[3], s2));
      p[1] = make_uint4(ptx::hmul2(b[0], s2), ptx::hmul2(b[1], s2), ptx::hmul2(b[2], s2), ptx::hmul2(b[3], s2));
      reinterpret_cast<uint32_t*>(dst + (long long)(i + u) * kExtRow + CKV)[lane] = any ? 0x7E007E00u : ptx::e4m3x2_to_f16x2(uint16_t(rp[u]));
    }
  }
}

__device__ __forceinline__ void ext_convert_rows(const ExtProblem& E, const ExtOperands& O, int item) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row0 = E.items[item].row0, rows = E.items[item].rows;
  const float ratio = O.kpe_scale / O.ckv_scale;  // rope scores in units of the latent ones
  for (int r = warp; r < kExtRows; r += kExtPrepThreads / 32) {
    const long long at = (long long)row0 + (r < rows ? r : rows - 1);  // (dead rows repeat the last live one and are not written out)
    const uint4* src = reinterpret_cast<const uint4*>(O.q_nope + at * CKV);
    const uint4 w0 = __ldg(src + lane), w1 = __ldg(src + 32 + lane);  // channels 8 lane .. of both halves of the row
    const uint32_t rp = __ldg(reinterpret_cast<const uint32_t*>(O.q_pe + at * KPE) + lane);
    const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
    const float p0 = __uint_as_float(rp << 16) * ratio, p1 = __uint_as_float(rp & 0xFFFF0000u) * ratio;
    uint32_t m = max(__float_as_uint(p0) & 0x7FFFFFFFu, __float_as_uint(p1) & 0x7FFFFFFFu);  // magnitudes, ordered like integers
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, max(w[j] << 16 & 0x7FFFFFFFu, w[j] & 0x7FFF0000u));
#pragma unroll
    for (int o = 16; o; o >>= 1) m = max(m, __shfl_xor_sync(~0u, m, o));
    int e = int(m >> 23) - 127 - 14;  // the row is held times 2^-e
    e = e < -100 ? -100 : e > 112 ? 112 : e;
    // the sign of the softmax scale goes into the row, so that a larger product is always a larger score
    const float up = (O.sm_scale_log2 < 0.f ? -1.f : 1.f) * __uint_as_float(uint32_t(127 - e) << 23);
    __half* const dst = O.q16 + ((long long)item * kExtRows + r) * kExtRow;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = ptx::f32x2_to_f16x2(__uint_as_float(w[4 * h + j] << 16) * up, __uint_as_float(w[4 * h + j] & 0xFFFF0000u) * up);
      reinterpret_cast<uint4*>(dst)[32 * h + lane] = make_uint4(o[0], o[1], o[2], o[3]);
    }
    reinterpret_cast<uint32_t*>(dst + CKV)[lane] = ptx::f32x2_to_f16x2(p0 * up, p1 * up);
    // (never 0: a masked score is -inf and must stay so; a row with a non-finite element is NaN)
    if (lane == 0)
      O.q_scale[(long long)item * kExtRows + r] =
          m < 0x7F800000u ? fmaxf(fabsf(O.sm_scale_log2) * O.ckv_scale * __uint_as_float(uint32_t(127 + e) << 23), 0x1p-149f) : __uint_as_float(0x7FC00000u);
  }
}

__global__ void __launch_bounds__(kExtPrepThreads) mla_extend_prep_kernel(const ExtProblem E, const ExtOperands O) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int first = E.indptr[0] < 0 ? 0 : E.indptr[0] < E.total_q ? E.indptr[0] : E.total_q;
  const int z = E.indptr[E.batch], last = z < first ? first : z < E.total_q ? z : E.total_q;
  const long long front = (long long)first * E.heads, none = front + (long long)(E.total_q - last) * E.heads;
  for (long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); i < none; i += (long long)gridDim.x * 4) {
    const long long row = i < front ? i : i - front + (long long)last * E.heads;
    O.out[row * (CKV / 8) + (threadIdx.x & 63)] = make_uint4(0, 0, 0, 0);
  }
  if (int(blockIdx.x) < E.max_tiles) {
    if (int(blockIdx.x) < E.counts[1]) ext_convert_tile(E, O, blockIdx.x);
  } else if (int(blockIdx.x) - E.max_tiles < E.counts[0]) {
    ext_convert_rows(E, O, int(blockIdx.x) - E.max_tiles);
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Merge of the partial results of an item that several pairs worked on: pair p holds its first tiles, the pairs behind it the rest. The
// partials of a pair: slot 2 p + 1 an item that it began, 2 p one that another pair began.
// ---------------------------------------------------------------------------------------------------------------
template <int GROUPS>
__global__ void __launch_bounds__(128 * GROUPS)
mla_extend_combine_kernel(const ExtProblem E, const float* __restrict__ lse_part, const float* __restrict__ o_part, void* out) {
  __shared__ float weights[kCombineMaxParts];
  __shared__ float4 partial[GROUPS > 1 ? (GROUPS - 1) * 128 : 1];
  ptx::grid_dependency_wait();
  const int p = blockIdx.x, r = blockIdx.y, item = E.pair[p].split;
  if (item < 0) return;
  const ExtItem& m = E.items[item];
  if (r >= m.rows) return;
  const int q = E.pair[1].first;  // tiles per pair (a split item has a second pair)
  const int parts = (m.prefix + m.ntiles - 1) / q - p + 1;
  auto slot = [&](int i) { return (long long)(i ? 2 * (p + i) : 2 * p + 1) * kExtRows + r; };
  merge_row<GROUPS>(
      parts, [&](int i) { return lse_part[slot(i)]; }, [&](int i) { return o_part + slot(i) * CKV; }, (long long)m.row0 + r, out, nullptr, nullptr,
      weights, partial);
}

}  // namespace mla
