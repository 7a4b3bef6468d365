// Chunks of new tokens, everything around the attention kernel (mla_extend_sm100.cuh): the schedule, the FP16 operands, the merge.
//
// The rows of a request (query token, head) are cut into tiles of 128, the ITEMS; an item's work is the 64-token BLOCKS of the cache
// that its rows see, four to a tile of the attention kernel. An item costs a pair its tiles and kItemCost more (its query, its output).
// The items are dealt out whole, item i to CTA pair i % pairs, for as many rounds as leave every pair at or below its even share of
// the cost; the tiles of the items that are left are laid end to end and cut so that every pair ends up with its share. Pairs that
// work at the same time thus work on neighbouring items, which read the same tokens. 24 ragged chunks of 16 heads (1 to 400 query
// tokens behind 0 to 8000 others, 115 MB of FP16 rows): 885 us; with shares of tiles alone 900; with one contiguous piece of the
// flattened tiles per pair 913 and 1.6 GB read from HBM (a third of the sectors missed L2).
//
// Window: the tokens that some query of the request sees are [0, S) and everything from the first query's window on. The cache is
// read into a numbering of blocks that has no gap: the first `sink_blocks` blocks, then the blocks from the window's on, `shift` tokens
// further in the request. An item skips the blocks between the first tokens' and its own window; its tiles are four of its blocks
// each, wherever these lie (with whole 256-token tiles, 8 windowed chunks of 4096 + 128 tokens took 18 tiles per item instead of 17).
//
// Operands: the attention kernel multiplies FP16. Every visible token is dequantised once per call into a workspace row of 576 (latent
// 512, rope 64, exact: e2m1 x e4m3 has six significant bits), every query row once into a row of the same shape, held times a power
// of two that puts its maximum into [2^14, 2^15) (latent elements are exact from 2^-31 of the maximum up and off by 2^-25 at most below) with the rope part times
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
constexpr int kExtBlock = 64;   // tokens of a block
constexpr int kExtTile = 256;   // tokens of a tile
constexpr int kExtRow = CKV + KPE;
constexpr int kExtMaxBatch = 2048;  // requests at a time
constexpr int kExtHeld = 1024;      // items whose tile counts the schedule keeps in shared memory
constexpr int kExtMaxPairs = 128;

struct alignas(16) ExtItem {  // (read and written in 16-byte words: as ints, 787 items took the schedule 12000 of its 26000 cycles)
  int prefix;      // tiles of the items before
  int ntiles;      // at least 1 (an item that sees nothing has one tile, all masked)
  int block0;      // first workspace block of the request
  int sinks, skip; // blocks: the first tokens' ones, and how many follow them that no row sees
  int shift;       // tokens: position of a token in the request minus its place in the request's workspace blocks, behind the first tokens' blocks
  int row0, rows;  // first row in [total_q * heads], number of rows
  int r0;          // first row within the request
  int pos0;        // position of the request's first query token
  int pad[2];
};
static_assert(sizeof(ExtItem) == 48, "ExtItem is three 16-byte words");

struct alignas(16) ExtPair {
  int rounds;              // whole items pair, pair + pairs, ...: this many
  int item, first, count;  // and of the rest: first item, first flattened tile, tiles
  int split, parts;        // item whose first tiles this pair holds and whose last ones another does, or -1; pairs that share it
  int pad[2];
};

// What the caller gives and how much room there is
struct ExtProblem {
  const int* kv_lens;
  const int* indptr;  // null: one query token per request
  int batch, total_q, heads, max_kv_len, window, sinks, pairs;
  int max_items, max_blocks;
  int first_q;      // without an indptr: index of the first request's query token
  int edges;        // 1: the rows in front of the first request's are this call's to fill with zeros, 2: those behind the last one's
  ExtItem* items;   // [max_items]
  ExtPair* pair;    // [pairs]
  int* status;
};

constexpr int kExtPrepThreads = 256;
// Costs in quarters of a tile. Measured, cycles: a tile 5900 to 6200, an item 10000 to 12500 beside its tiles.
constexpr int kTileCost = 4, kItemCost = 7;

// inclusive scan over a block of WARPS warps (every thread takes part); `sums`: 32 of them; the block's sum in `all`
template <int WARPS, class T>
__device__ __forceinline__ T block_scan(T v, long long* held, T& all) {
  T* sums = reinterpret_cast<T*>(held);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T u = __shfl_up_sync(~0u, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    T w = lane < WARPS ? sums[lane] : T(0);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T u = __shfl_up_sync(~0u, w, o);
      if (lane >= o) w += u;
    }
    sums[lane] = w;
  }
  __syncthreads();
  all = sums[31];
  return v + (warp ? sums[warp - 1] : T(0));
}

struct ExtRequest {
  int q0, q, n, pos0, begin, shift, sink_blocks, blocks;
};
// index of request b's first query token; without an indptr every request has one
__device__ __forceinline__ int ext_first(const ExtProblem& E, int b) { return E.indptr ? E.indptr[b] : E.first_q + b; }
__device__ __forceinline__ int ext_blocks(int tokens) { return int((uint32_t(tokens) + kExtBlock - 1) / kExtBlock); }  // (not negative)
__device__ __forceinline__ ExtRequest ext_request(const ExtProblem& E, int b) {
  ExtRequest r;
  const int a = ext_first(E, b), z = ext_first(E, b + 1);
  const int lo = a < 0 ? 0 : a, hi = z < E.total_q ? z : E.total_q;
  r.q0 = lo, r.q = hi > lo ? hi - lo : 0;
  const int n = E.kv_lens[b];
  r.n = n < 0 ? 0 : n < E.max_kv_len ? n : E.max_kv_len;
  r.pos0 = r.q ? r.n - (z - lo) : 0;  // (z > lo >= 0)
  r.shift = 0, r.sink_blocks = 0, r.begin = 0;
  if (E.window > 0) {
    const long long s = ((long long)E.sinks + kExtBlock - 1) / kExtBlock;
    const long long begin = (long long)r.pos0 - E.window + 1;  // first token in the window of the first query token
    r.begin = begin > 0 ? int(begin) : 0;
    const long long t = r.begin / kExtBlock;
    if (t > s) r.shift = int(t - s) * kExtBlock;
    r.sink_blocks = int(s < ext_blocks(r.n) ? s : ext_blocks(r.n));
  }
  r.blocks = ext_blocks(r.n - r.shift);
  if (r.blocks < 1) r.blocks = 1;
  if (r.q == 0) r.blocks = 0;
  return r;
}

// Where the requests' items and workspace blocks begin. Every CTA of the call's first kernel works this out for itself: the first one
// makes the schedule, the others convert operands meanwhile (32 windowed single tokens of 128 heads: 66.7 us one after the other, 61.3 so; 24 to
// 33 us of small calls 1 to 2 less than with a launch of its own for the schedule).
struct ExtTables {
  int item0[kExtMaxBatch], block0[kExtMaxBatch];  // items and blocks of the requests before
  long long sums[32];
  int items, blocks;
  bool failed;  // there is no room for what the query index asks for: no items, and zeros in the output
};
__device__ __forceinline__ void ext_tables(const ExtProblem& E, ExtTables& s) {
  constexpr int THREADS = kExtPrepThreads;
  const int tid = threadIdx.x;
  // A query index that runs backwards or past total_q could ask for more than there is room for. A request has less than 2^26 of
  // either, so that a round's 256 requests may add up to 2^34: sums of 64 bits, and no further round after one without room. Ordinary
  // counts share one sum (two of 64 bits each time: 32 windowed single tokens of 128 heads 62.3 us instead of 62.0).
  int items = 0, blocks = 0;
  bool failed = false;
  for (int b0 = 0; b0 < E.batch; b0 += THREADS) {
    const int b = b0 + tid;
    long long mine = 0, ii, ib, all_items, all_blocks;
    ExtRequest r = {};
    if (b < E.batch) {
      r = ext_request(E, b);
      mine = ((long long)r.q * E.heads + kExtRows - 1) / kExtRows;
    }
    if (!__syncthreads_or(mine >= 1 << 22 || r.blocks >= 1 << 22)) {  // the sums are below 2^30
      long long all;
      const long long both = mine << 32 | r.blocks, at = block_scan<THREADS / 32>(both, s.sums, all) - both;
      ii = at >> 32, ib = uint32_t(at), all_items = all >> 32, all_blocks = uint32_t(all);
    } else {
      ii = block_scan<THREADS / 32>(mine, s.sums, all_items) - mine;
      ib = block_scan<THREADS / 32>((long long)r.blocks, s.sums, all_blocks) - r.blocks;
    }
    ii += items, ib += blocks;
    failed = items + all_items > E.max_items || blocks + all_blocks > E.max_blocks;
    if (failed) break;
    items += int(all_items), blocks += int(all_blocks);
    if (b < E.batch) s.item0[b] = int(ii), s.block0[b] = int(ib);
  }
  if (failed && tid == 0 && E.status) atomicExch(E.status, int(kBadSchedule));
  if (tid == 0) s.items = failed ? 0 : items, s.blocks = failed ? 0 : blocks, s.failed = failed;
  __syncthreads();
}

__device__ __forceinline__ void ext_schedule(const ExtProblem& E, ExtTables& tab) {
  __shared__ int2 held[kExtHeld];        // {prefix, tiles} of an item
  __shared__ int cut[kExtMaxPairs + 1];  // tiles of the rest before pair p
  __shared__ int rounds_s;
  const int tid = threadIdx.x;
  constexpr int kWarps = kExtPrepThreads / 32;
  static_assert(kExtMaxPairs <= kExtPrepThreads, "a thread per pair");
  const int items = tab.items;
  if (tid == 0) rounds_s = items / E.pairs;

  // ---- items
  int total = 0;
  for (int i0 = 0; i0 < items; i0 += kExtPrepThreads) {
    const int i = i0 + tid;
    ExtItem m = {};
    if (i < items) {
      int lo = 0, hi = E.batch - 1;  // last b with item0[b] <= i
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.item0[mid] <= i) lo = mid;
        else hi = mid - 1;
      }
      const ExtRequest r = ext_request(E, lo);
      m.r0 = (i - tab.item0[lo]) * kExtRows;
      const long long rows = (long long)r.q * E.heads - m.r0;
      m.rows = int(rows < kExtRows ? rows : kExtRows);
      m.row0 = r.q0 * E.heads + m.r0, m.pos0 = r.pos0, m.shift = r.shift, m.block0 = tab.block0[lo];
      const int first = r.pos0 + m.r0 / E.heads, last = r.pos0 + (m.r0 + m.rows - 1) / E.heads;  // positions of its query tokens
      const int end = last + 1 < r.n ? last + 1 : r.n;                                           // tokens before it are seen
      int e = end > r.shift ? ext_blocks(end - r.shift) : 0;                                     // blocks up to there
      if (E.window > 0) {
        const long long begin = (long long)first - E.window + 1 - r.shift;
        const int t = begin > 0 ? int(begin / kExtBlock) : 0;
        m.sinks = r.sink_blocks;
        if (t > m.sinks) m.skip = t - m.sinks;
      }
      if (e > r.blocks) e = r.blocks;
      m.ntiles = (e - m.skip + kExtTile / kExtBlock - 1) / (kExtTile / kExtBlock);
      if (m.ntiles < 1) m.ntiles = 1, m.skip = 0;
    }
    int all;
    const int incl = block_scan<kWarps>(m.ntiles, tab.sums, all);
    if (i < items) {
      m.prefix = total + incl - m.ntiles;
      E.items[i] = m;
      if (i < kExtHeld) held[i] = make_int2(m.prefix, m.ntiles);
    }
    total += all;
  }
  __syncthreads();
  auto tiles_of = [&](int i) { return i < kExtHeld ? held[i] : make_int2(E.items[i].prefix, E.items[i].ntiles); };

  // ---- rounds of whole items
  const long long cost = (long long)kTileCost * total + (long long)kItemCost * items;
  const long long share = (cost + E.pairs - 1) / E.pairs;
  const int most = items / E.pairs;
  constexpr int kAhead = 8;  // loads in flight
  auto load_after = [&](int rounds, long long limit, int& fits) {  // cost of this pair's first `rounds` items; how many of them stay within `limit`
    long long sum = 0;
    fits = 0;
    for (int k = 0; k < rounds; k += kAhead) {
      int n[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) n[j] = k + j < rounds ? tiles_of(tid + (k + j) * E.pairs).y : 0;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (k + j < rounds) sum += kTileCost * n[j] + kItemCost;
        if (k + j < rounds && sum <= limit) fits = k + j + 1;
      }
    }
    return sum;
  };
  int fits;
  long long load = 0;
  if (tid < E.pairs) {
    load = load_after(most, share, fits);
    if (fits < most) atomicMin(&rounds_s, fits);
  }
  __syncthreads();
  const int rounds = rounds_s;
  if (tid < E.pairs && rounds < most) load = load_after(rounds, share, fits);
  // ---- the rest: cut at the pairs' remaining shares
  const int rest0 = rounds * E.pairs;                                       // first item of the rest
  const int base = rest0 < items ? tiles_of(rest0).x : total, rest = total - base;
  const long long room = tid < E.pairs ? share - load : 0;
  long long all;
  const long long at = block_scan<kWarps>(room, tab.sums, all) - room;
  if (tid < E.pairs) {
    // the tile of the rest at cost `at`: in item i at cost c(i) = kTileCost * tiles before it + kItemCost * items before it
    int lo = rest0, hi = items - 1;  // last item with c(i) <= at
    auto c = [&](int i) { return (long long)kTileCost * (tiles_of(i).x - base) + (long long)kItemCost * (i - rest0); };
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (c(mid) <= at) lo = mid;
      else hi = mid - 1;
    }
    int tile = rest;
    if (lo < items) {
      const int2 it = tiles_of(lo);
      const long long in = (at - c(lo) - kItemCost + kTileCost / 2) / kTileCost;  // (nearest)
      tile = it.x - base + int(in < 0 ? 0 : in < it.y ? in : it.y);
    }
    cut[tid] = tid == 0 ? 0 : tile < rest ? tile : rest;
    if (tid == 0) cut[E.pairs] = rest;
  }
  __syncthreads();
  if (tid < E.pairs) {
    ExtPair o = {rounds, 0, base + cut[tid], cut[tid + 1] - cut[tid], -1, 0, {0, 0}};
    E.pair[tid] = o;
  }
  __syncthreads();
  for (int i = rest0 + tid; i < items; i += kExtPrepThreads) {
    const int2 it = tiles_of(i);
    const int a = it.x - base, z = a + it.y;
    auto holder = [&](int x) {  // last pair whose piece starts at or before tile x (pieces without tiles lie in front of it)
      int lo = 0, hi = E.pairs - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cut[mid] <= x) lo = mid;
        else hi = mid - 1;
      }
      return lo;
    };
    const int p0 = holder(a), p1 = holder(z - 1);
    for (int p = cut[p0] == a ? p0 : p0 + 1; p <= p1; ++p)
      if (cut[p + 1] > cut[p]) E.pair[p].item = i;
    if (p1 > p0) E.pair[p0].split = i, E.pair[p0].parts = p1 - p0 + 1;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Operands. A unit of work is a block of 64 tokens or 32 rows of an item, 8 or 4 per warp: all loads of a warp's four rows are
// issued before the first is used. All blocks share the rows of no request (zeros in the output).
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
  __half* kv16;     // [max_blocks * 64][576]
  __half* q16;      // [max_items * 128][576]
  float* q_scale;   // [max_items * 128]: factor of a row's scores, log2 units
  uint4* out;       // [total_q * heads][512] BF16
};

constexpr int kExtQRows = 32;   // rows of a unit

// last b in [0, n) with a[b] <= x (a is non-decreasing, a[0] <= x), by the whole warp: 32 probes at a time
__device__ __forceinline__ int warp_upper(const int* a, int n, int x) {
  const int lane = threadIdx.x & 31;
  int lo = 0;
  while (n > 1) {
    const int step = (n + 31) >> 5, i = lo + lane * step;
    const uint32_t below = __ballot_sync(~0u, lane * step < n && a[i] <= x);  // a prefix of the lanes, lane 0 in it
    const int k = 31 - __clz(below);
    lo += k * step, n = n - k * step < step ? n - k * step : step;
  }
  return lo;
}

__device__ __forceinline__ void ext_convert_tokens(const ExtProblem& E, const ExtOperands& O, const ExtTables& tab, int unit) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kPer = kExtBlock / (kExtPrepThreads / 32);  // tokens of a warp
  const int t0 = unit * kExtBlock + kPer * warp;
  const int lo = warp_upper(tab.block0, E.batch, unit);
  const ExtRequest r = ext_request(E, lo);
  const int v = t0 - tab.block0[lo] * kExtBlock + lane;  // this lane's token among the request's
  int src = -1;                                          // its cache row; -1: zeros
  if (lane < kPer && v < r.n - r.shift && unit < tab.blocks) {
    const int tok = v < r.sink_blocks * kExtBlock ? v : v + r.shift;
    // (tokens between the first ones and the window belong to blocks that are read, but their pages may be gone)
    if (tok < E.sinks || tok >= r.begin) {
      const int pi = tok >> O.page_shift;
      const int page = pi < O.pt_width ? O.page_table[(long long)lo * O.pt_stride + pi] : -1;
      if (page >= 0 && page < O.num_pages) src = (page << O.page_shift) + (tok & ((1 << O.page_shift) - 1));
      else if (E.status) atomicExch(E.status, int(kBadPage));
    }
  }
  __half* const dst = O.kv16 + (long long)t0 * kExtRow;
  constexpr int U = 4;
#pragma unroll
  for (int i = 0; i < kPer; i += U) {
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

__device__ __forceinline__ void ext_convert_rows(const ExtProblem& E, const ExtOperands& O, const ExtTables& tab, int unit) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int item = unit / (kExtRows / kExtQRows);
  constexpr int U = kExtQRows / (kExtPrepThreads / 32);  // rows of a warp
  const int r0 = (unit % (kExtRows / kExtQRows)) * kExtQRows + U * warp;
  const int b = warp_upper(tab.item0, E.batch, item), first = (item - tab.item0[b]) * kExtRows;  // of the request's rows
  const ExtRequest r = ext_request(E, b);
  const long long row0 = (long long)r.q0 * E.heads + first, rows = (long long)r.q * E.heads - first;  // (of which the item has up to 128)
  const float ratio = O.kpe_scale / O.ckv_scale;  // rope scores in units of the latent ones
  uint4 w0[U], w1[U];
  uint32_t rp[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long at = row0 + (r0 + u < rows ? r0 + u : rows - 1);  // (dead rows repeat the last live one and are not written out)
    const uint4* src = reinterpret_cast<const uint4*>(O.q_nope + at * CKV);
    w0[u] = __ldg(src + lane), w1[u] = __ldg(src + 32 + lane);  // channels 8 lane .. of both halves of the row
    rp[u] = __ldg(reinterpret_cast<const uint32_t*>(O.q_pe + at * KPE) + lane);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t w[8] = {w0[u].x, w0[u].y, w0[u].z, w0[u].w, w1[u].x, w1[u].y, w1[u].z, w1[u].w};
    const float p0 = __uint_as_float(rp[u] << 16) * ratio, p1 = __uint_as_float(rp[u] & 0xFFFF0000u) * ratio;
    uint32_t m = max(__float_as_uint(p0) & 0x7FFFFFFFu, __float_as_uint(p1) & 0x7FFFFFFFu);  // magnitudes, ordered like integers
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, max(w[j] << 16 & 0x7FFFFFFFu, w[j] & 0x7FFF0000u));
    m = __reduce_max_sync(~0u, m);
    int e = int(m >> 23) - 127 - 14;  // the row is held times 2^-e
    e = e < -100 ? -100 : e > 112 ? 112 : e;
    // the sign of the softmax scale goes into the row, so that a larger product is always a larger score
    const float up = (O.sm_scale_log2 < 0.f ? -1.f : 1.f) * __uint_as_float(uint32_t(127 - e) << 23);
    __half* const dst = O.q16 + ((long long)item * kExtRows + r0 + u) * kExtRow;
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
      O.q_scale[(long long)item * kExtRows + r0 + u] =
          m < 0x7F800000u ? fmaxf(fabsf(O.sm_scale_log2) * O.ckv_scale * __uint_as_float(uint32_t(127 + e) << 23), 0x1p-149f) : __uint_as_float(0x7FC00000u);
  }
}

// The first CTA makes the schedule, the others the operands.
__global__ void __launch_bounds__(kExtPrepThreads) mla_extend_prep_kernel(const ExtProblem E, const ExtOperands O) {
  __shared__ ExtTables tab;
  ptx::grid_launch_dependents();
  ext_tables(E, tab);
  if (blockIdx.x == 0) {
    ext_schedule(E, tab);
    return;
  }
  const int cta = int(blockIdx.x) - 1, ctas = int(gridDim.x) - 1;
  const int a = ext_first(E, 0), first = a < 0 ? 0 : a < E.total_q ? a : E.total_q;
  const int z = ext_first(E, E.batch), last = z < first ? first : z < E.total_q ? z : E.total_q;
  // query tokens [a0, a1) and [b0, b1) get zeros: those of no request, or all of the call's requests where they find no room
  const int a0 = E.edges & 1 ? 0 : first, a1 = tab.failed ? last : first, b0 = last, b1 = E.edges & 2 ? E.total_q : last;
  const long long front = (long long)(a1 - a0) * E.heads, none = front + (long long)(b1 - b0) * E.heads;
  for (long long i = (long long)cta * 4 + (threadIdx.x >> 6); i < none; i += (long long)ctas * 4) {
    const long long row = i < front ? i + (long long)a0 * E.heads : i - front + (long long)b0 * E.heads;
    O.out[row * (CKV / 8) + (threadIdx.x & 63)] = make_uint4(0, 0, 0, 0);
  }
  if (tab.failed) return;
  // (the last tile reads up to three blocks behind the last one, with weight 0: zeros)
  const int tokens = tab.blocks + 3 < E.max_blocks ? tab.blocks + 3 : E.max_blocks, units = tokens + tab.items * (kExtRows / kExtQRows);
  for (int i = cta; i < units; i += ctas) {
    if (i < tokens) ext_convert_tokens(E, O, tab, i);
    else ext_convert_rows(E, O, tab, i - tokens);
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Merge of the partial results of an item that several pairs worked on: pair p holds its first tiles, the pairs behind it the rest. The
// partials of a pair: slot 2 p + 1 an item that it began, 2 p one that another pair began. A warp takes a row, two partials at a time
// (eight 16-byte loads per lane in flight).
// ---------------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(128, 8)
mla_extend_combine_kernel(const ExtProblem E, const float* __restrict__ lse_part, const float* __restrict__ o_part, uint2* __restrict__ out) {
  ptx::grid_dependency_wait();
  const int p = blockIdx.x, lane = threadIdx.x & 31;
  const ExtPair pair = E.pair[p];
  if (pair.split < 0) return;
  const int row0 = E.items[pair.split].row0, rows = E.items[pair.split].rows, parts = pair.parts;
  const int r = 4 * blockIdx.y + (threadIdx.x >> 5);
  if (r >= rows) return;
  auto slot = [&](int i) { return (long long)(i ? 2 * (p + i) : 2 * p + 1) * kExtRows + r; };
  // the weights, one partial per lane and round (a pair may have got none of the rest: nothing is in its slot)
  constexpr int kRounds = (kExtMaxPairs + 31) / 32;
  float w[kRounds], M = -INFINITY, den = 0.f;
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int i = 32 * k + lane;
    w[k] = i < parts && (i == 0 || E.pair[p + i].count > 0) ? lse_part[slot(i)] : -INFINITY;
    M = fmaxf(M, w[k]);
  }
  M = warp_max(M);
#pragma unroll
  for (int k = 0; k < kRounds; ++k) w[k] = w[k] == -INFINITY ? 0.f : exp2f(w[k] - M), den += w[k];
  den = warp_sum(den);
  float4 acc[4] = {};
  auto add = [&](float wi, const float4 (&v)[4]) {
    if (wi == 0.f) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j].x += wi * v[j].x, acc[j].y += wi * v[j].y, acc[j].z += wi * v[j].z, acc[j].w += wi * v[j].w;
  };
  constexpr int U = 2;  // partials in flight
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    for (int i = 0; i < 32 && 32 * k + i < parts; i += U) {
      float wi[U];
      float4 v[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        wi[u] = __shfl_sync(~0u, w[k], i + u);
        const float4* src = reinterpret_cast<const float4*>(o_part + slot(32 * k + i + u) * CKV) + lane;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[u][j] = wi[u] != 0.f ? src[32 * j] : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) add(wi[u], v[u]);
    }
  }
  const float s = den != 0.f ? 1.f / den : 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    out[((long long)row0 + r) * (CKV / 4) + 32 * j + lane] = make_uint2(pack_bf16x2(acc[j].x * s, acc[j].y * s), pack_bf16x2(acc[j].z * s, acc[j].w * s));
}

}  // namespace mla
