// Attention of a chunk of new tokens over the paged latent cache, 16-bit mode, on PAIRS of CTAs that share every MMA
// (tcgen05 cta_group::2, M = 128 rows, 64 per CTA). The operands are FP16 rows that the call's first kernels wrote (mla_extend_prep.cuh).
//
//   QK^T : S[row, token] = Q[row, 576] . K^T    A = Q (smem, 64 rows per CTA), B = K: CTA c holds tokens [128 c, +128) of a 256-token
//                                               tile; N = 256, 36 K steps
//   PV   : O[row, chan] += P[row, token] . V    A = P (smem, FP16), B = V read MN-major: CTA c holds channels 256 i + [128 c, +128) of all
//                                               256 tokens; N = 256 channels, i = 0, 1, 16 K steps each
//
// O of 128 rows x 512 channels in fp32 fills a CTA's tensor memory. With 64 rows per CTA it takes half (lanes 0..63: channels
// 256 i + [0, 128), lanes 64..127: the next 128), and both S buffers the other half: QK^T of tile g + 1 runs while the softmax of tile g
// does. As the pair shares B, each CTA loads half of it; K is split by tokens and V by channels, so a token row crosses into
// shared memory twice (its K part in one CTA, halves of its V part in both): 278 KB per tile and CTA.
//
// What bounds it: the tensor pipe needs 36 * 64 + 32 * 64 = 4352 cycles per tile, shared memory 5690 (728 KB at 128 bytes per cycle: A and
// B of the products 408, the loads 278, P 32; measured 5900 to 6200), and in calls of more than a few hundred us the 1 kW power
// limit holds the clock at 1.55 to 1.62 GHz. 1024 query tokens of 128 heads behind 15360 others: 3.56 ms, 1.27 PFLOP/s, 0.93 of what the
// library's BF16 product sustains; 4 chunks of 512 of 16 heads behind 7680: 418 us of the call's 484, tensor pipe 73 % busy (ncu),
// 76 MB from HBM, 10.7 TB/s from L2. The end of an item costs a pair 10000 to 12500 cycles (output, next query, pipeline filling).
// Stalls that were taken out without the time changing, which is how the power limit shows: a thread of its own for the query's
// loads, output by four more warps, output straight from registers, the query converted in here. M = 256 per pair (two thirds of the
// shared-memory traffic per row) would need all of tensor memory for O.
//
// Tensor memory: O: 0..255 | S: 256..511 (two buffers of 128).
// Shared memory: Q 72 KB | P 32 KB | ring of seven 16 KB units (K: 128 tokens x 64 channels; V: 64 tokens x 128 channels).
// Warp roles (384 threads): 0-7 softmax + epilogue, 8 TMA producer, 9 MMA issue (rank 0), 10 tensor memory. Every wait is bounded.
#pragma once
#include <cuda_fp16.h>
#include "mla_extend_prep.cuh"
#include "ptx_sm100.cuh"

namespace mla {

constexpr int kExtThreads = 384;
constexpr int kExtUnits = 7;             // ring units
constexpr int kExtPanel = 64 * 128;      // 64 rows x 64 channels, 128-byte swizzle
constexpr int kExtUnit = 2 * kExtPanel;  // K: 128 tokens x 64 channels (token halves one behind the other); V: 64 tokens x two 64-channel panels

struct ExtSmem {
  alignas(1024) uint8_t q[9][kExtPanel];
  alignas(1024) uint8_t p[4][kExtPanel];  // 64 rows x 64 tokens
  alignas(1024) uint8_t ring[kExtUnits][kExtUnit];
  float xch[4][64], xl[4][64];             // maxima / sums of a row's four threads
  // in rank 0: counted by both CTAs
  alignas(8) uint64_t full[kExtUnits], q_full, s_free[2], p_full, o_free;
  // in both: MMA completion
  uint64_t empty[kExtUnits], q_empty, s_full[2], pv_done;
  uint32_t tmem_base;
  int abort_flag;
};
constexpr size_t ext_smem_bytes() { return sizeof(ExtSmem) + 1024; }
static_assert(ext_smem_bytes() <= 232448, "chunk attention kernel exceeds the shared memory a CTA can opt in to");

struct ExtCols {
  static constexpr uint32_t O = 0, S = 256;
};

// The pair's tiles, item by item: tiles [t0, t1) of `item`, whole items first. Every role walks through the same sequence.
struct ExtWalk {
  const ExtProblem& E;
  int rounds, left, at, next_item, round_item, item;
  __device__ __forceinline__ ExtWalk(const ExtProblem& e, int pair) : E(e) {
    const ExtPair p = e.pair[pair];
    rounds = p.rounds, left = p.count, at = p.first, next_item = p.item, round_item = pair, item = 0;
  }
  __device__ __forceinline__ bool next(ExtItem& m, int& t0, int& t1) {
    if (rounds > 0) {
      --rounds, item = round_item, round_item += E.pairs;
      m = E.items[item];
      t0 = 0, t1 = m.ntiles;
      return true;
    }
    if (left <= 0) return false;
    item = next_item++;
    m = E.items[item];
    t0 = at - m.prefix;
    t1 = m.ntiles - t0 < left ? m.ntiles : t0 + left;
    left -= t1 - t0, at += t1 - t0;
    return true;
  }
};
// workspace block of block j of an item, within the request (blocks behind the item's last are read and masked)
__device__ __forceinline__ int ext_block(const ExtItem& m, int j) { return j < m.sinks ? j : j + m.skip; }

struct ExtParams {
  ExtProblem E;
  const float* q_scale;
  float ckv_scale;
  float* lse_part;  // [2 * pairs][128]
  float* o_part;    // [2 * pairs][128][512]
  uint16_t* out;    // BF16
  int* status;
};

// ---------------------------------------------------------------------------------------------------------------
// role: TMA producer (one thread per CTA). Units in the order in which the MMAs take them: K of tile g, then V of tile g - 1.
// ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void ext_producer_role(ExtSmem& s, const ExtParams& P, const CUtensorMap* kv_map, const CUtensorMap* q_map, int pair,
                                                  uint32_t rank) {
  const uint32_t ring = ptx::smem_u32(s.ring[0]), q = ptx::smem_u32(s.q[0]);
  const uint32_t full0 = ptx::map_to_cta(&s.full[0], 0), q_full = ptx::map_to_cta(&s.q_full, 0);
  uint32_t slot = 0, phase = 1;  // of the next ring unit; parity of the wait for it to be free
  // two boxes of 64 rows x 64 channels into the next unit
  auto load = [&](int x0, int y0, int x1, int y1) {
    if (!ptx::mbar_wait(&s.empty[slot], phase, &s.abort_flag)) return false;
    if (rank == 0) ptx::mbar_arrive_expect_tx(&s.full[slot], 2 * kExtUnit);
    ptx::tma_load_2d_pair(ring + slot * kExtUnit, kv_map, x0, y0, full0 + 8 * slot);
    ptx::tma_load_2d_pair(ring + slot * kExtUnit + kExtPanel, kv_map, x1, y1, full0 + 8 * slot);
    if (++slot == kExtUnits) slot = 0, phase ^= 1;
    return true;
  };
  auto load_k = [&](const int (&row)[4]) {
    const int y0 = rank ? row[2] : row[0], y1 = rank ? row[3] : row[1];
#pragma unroll 1
    for (int u = 0; u < 9; ++u)
      if (!load(64 * u, y0, 64 * u, y1)) return false;
    return true;
  };
  auto load_v = [&](const int (&row)[4]) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {  // block u / 2, channel half u % 2
      const int x = 256 * (u & 1) + 128 * int(rank);
      if (!load(x, row[u >> 1], x + 64, row[u >> 1])) return false;
    }
    return true;
  };
  ExtWalk walk(P.E, pair);
  ExtItem m;
  int t0, t1, before[4] = {-1, -1, -1, -1};  // workspace rows of the blocks of the tile whose V is due
  uint32_t n_items = 0;
  while (walk.next(m, t0, t1)) {
    // the query, once every QK^T of the item before has read the old one
    if (!ptx::mbar_wait(&s.q_empty, (n_items & 1) ^ 1, &s.abort_flag)) return;
    if (rank == 0) ptx::mbar_arrive_expect_tx(&s.q_full, 2 * 9 * kExtPanel);
#pragma unroll 1
    for (int p = 0; p < 9; ++p) ptx::tma_load_2d_pair(q + p * kExtPanel, q_map, 64 * p, walk.item * kExtRows + 64 * int(rank), q_full);
    ++n_items;
    for (int t = t0; t < t1; ++t) {
      int row[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) row[j] = (m.block0 + ext_block(m, 4 * t + j)) * kExtBlock;
      if (!load_k(row)) return;
      if (before[0] >= 0 && !load_v(before)) return;
#pragma unroll
      for (int j = 0; j < 4; ++j) before[j] = row[j];
    }
  }
  if (before[0] >= 0) load_v(before);
}

// ---------------------------------------------------------------------------------------------------------------
// role: MMA issue (one thread of rank 0): QK^T of tile g, then PV of tile g - 1
// ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void ext_mma_role(ExtSmem& s, const ExtParams& P, int pair) {
  const uint32_t tm = 0;  // all 512 columns are allocated: they start at column 0
  const uint32_t qk_desc = ptx::instr_desc(kExtRows, kExtTile, ptx::FMT_F16, ptx::FMT_F16, false, false);
  const uint32_t pv_desc = ptx::instr_desc(kExtRows, 256, ptx::FMT_F16, ptx::FMT_F16, false, true);
  const uint64_t q_d = ptx::smem_desc_sw128(ptx::smem_u32(s.q[0]), 16, 1024), p_d = ptx::smem_desc_sw128(ptx::smem_u32(s.p[0]), 16, 1024);
  const uint64_t k_d = ptx::smem_desc_sw128(ptx::smem_u32(s.ring[0]), 16, 1024);
  const uint64_t v_d = ptx::smem_desc_sw128(ptx::smem_u32(s.ring[0]), kExtPanel, 1024);  // channels 64 .. of the unit are a panel further
  const uint32_t hi = uint32_t(q_d >> 32), v_hi = uint32_t(v_d >> 32);
  uint32_t slot = 0, phase = 0, n_items = 0;
  auto advance = [&] {
    ptx::mma_commit_pair(&s.empty[slot]);
    if (++slot == kExtUnits) slot = 0, phase ^= 1;
  };
  bool first_of_item = false;
  auto pv = [&](uint32_t g, bool first, uint32_t segment) {
    if (!ptx::mbar_wait(&s.p_full, g & 1, &s.abort_flag)) return false;
    // a new item's first product overwrites O: the one before must have been read out
    if (first && segment > 0 && !ptx::mbar_wait(&s.o_free, (segment - 1) & 1, &s.abort_flag)) return false;
#pragma unroll 1
    for (int u = 0; u < 8; ++u) {
      if (!ptx::mbar_wait(&s.full[slot], phase, &s.abort_flag)) return false;
      ptx::tc_fence_after_sync();
      const uint32_t a = uint32_t(p_d) + (u >> 1) * (kExtPanel >> 4), b = uint32_t(v_d) + slot * (kExtUnit >> 4);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        ptx::mma_pair_f16_ss_lo(tm + ExtCols::O + 128 * (u & 1), a + 2 * ks, b + ks * (16 * 128 >> 4), hi, v_hi, pv_desc, !first || u > 1 || ks > 0);
      advance();
    }
    ptx::mma_commit_pair(&s.pv_done);
    return true;
  };
  ExtWalk walk(P.E, pair);
  ExtItem m;
  int t0, t1;
  uint32_t g = 0;
  while (walk.next(m, t0, t1)) {
    if (!ptx::mbar_wait(&s.q_full, n_items & 1, &s.abort_flag)) return;
    for (int t = t0; t < t1; ++t, ++g) {
      // the softmax warps of both CTAs have read the scores of tile g - 2
      if (g >= 2 && !ptx::mbar_wait(&s.s_free[g & 1], ((g >> 1) - 1) & 1, &s.abort_flag)) return;
      ptx::tc_fence_after_sync();
      const uint32_t d = tm + ExtCols::S + 128 * (g & 1);
#pragma unroll 1
      for (int u = 0; u < 9; ++u) {
        if (!ptx::mbar_wait(&s.full[slot], phase, &s.abort_flag)) return;
        ptx::tc_fence_after_sync();
        const uint32_t a = uint32_t(q_d) + u * (kExtPanel >> 4), b = uint32_t(k_d) + slot * (kExtUnit >> 4);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) ptx::mma_pair_f16_ss_lo(d, a + 2 * ks, b + 2 * ks, hi, hi, qk_desc, (u | ks) != 0);
        advance();
      }
      ptx::mma_commit_pair(&s.s_full[g & 1]);
      if (t + 1 == t1) ptx::mma_commit_pair(&s.q_empty);
      // PV of the tile before: in this item, or the last one of the item before
      if (g > 0 && !pv(g - 1, first_of_item, t > t0 ? n_items : n_items - 1)) return;
      first_of_item = t == t0;
    }
    ++n_items;
  }
  if (g > 0) pv(g - 1, first_of_item, n_items - 1);
}

// ---------------------------------------------------------------------------------------------------------------
// role: softmax + epilogue (8 warps). Warp w: lane quadrant w % 4, half w / 4. A row of the CTA's 64 has four threads: quadrants q and
// q + 2 (tokens 0..127 and 128..255 of a tile, of O the lower and upper 128 channels of each half), halves 0 and 1 (64 of
// these tokens; channels [256 half, +256)). The four warps of 32 rows keep a common running maximum: they vote once per tile and exchange
// maxima only when some row outgrows its own by 2^8.
// ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void ext_softmax_role(ExtSmem& s, const ExtParams& P, int pair, uint32_t rank) {
  const int lane = ptx::lane_id(), warp = threadIdx.x >> 5;
  const int quad = warp & 3, half = warp >> 2, part = 2 * (quad >> 1) + half;
  const int h = 32 * (quad & 1) + lane;  // row of the CTA
  const uint32_t tm_lane = s.tmem_base + (uint32_t(32 * quad) << 16);
  const uint32_t bar = 1 + (quad & 1);
  const uint32_t s_free0 = ptx::map_to_cta(&s.s_free[0], 0), p_full = ptx::map_to_cta(&s.p_full, 0), o_free = ptx::map_to_cta(&s.o_free, 0);
  const uint32_t p_row = ptx::smem_u32(s.p[part]) + h * 128;
  constexpr float kGrow = 8.f;
  ExtWalk walk(P.E, pair);
  ExtItem m;
  int t0, t1;
  uint32_t g = 0;
  while (walk.next(m, t0, t1)) {
    const int r = 64 * int(rank) + h;  // row of the item
    // the row sees tokens [begin, end) and [0, sinks)
    const int pos = m.pos0 + (m.r0 + (r < m.rows ? r : m.rows - 1)) / P.E.heads;
    const int end = pos + 1;
    const float qa = end > 0 ? P.q_scale[(long long)walk.item * kExtRows + r] : 1.f;  // (a row that sees nothing is 0 even if its query is not finite)
    const int begin = P.E.window > 0 && end > P.E.window ? end - P.E.window : 0, sinks = P.E.window > 0 ? P.E.sinks : 0;
    float mx_run = -INFINITY, l = 0.f;  // the maximum is the same in the row's four threads; l is this thread's share of the sum
    for (int t = t0; t < t1; ++t, ++g) {
      const uint32_t buf = g & 1;
      const bool ok = ptx::mbar_wait(&s.s_full[buf], (g >> 1) & 1, &s.abort_flag);
      ptx::tc_fence_after_sync();
      uint32_t sr[64];
      if (ok) {
        uint32_t (&lo)[32] = reinterpret_cast<uint32_t (&)[32]>(sr[0]);
        uint32_t (&hi)[32] = reinterpret_cast<uint32_t (&)[32]>(sr[32]);
        ptx::tmem_ld32(tm_lane + ExtCols::S + 128 * buf + 64 * half, lo);
        ptx::tmem_ld32(tm_lane + ExtCols::S + 128 * buf + 64 * half + 32, hi);
        ptx::tmem_wait_ld();
      }
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cta(s_free0 + 8 * buf);
      // position of this thread's first token
      const int j = 4 * t + part, at = ext_block(m, j) * kExtBlock + (j < m.sinks ? 0 : m.shift);
      const int hi_t = end - at, lo_t = begin - at, sk_t = sinks - at;
      if (!ok || hi_t < 64 || (lo_t > 0 && sk_t < 64)) {
#pragma unroll
        for (int k = 0; k < 64; ++k) sr[k] = ok && k < hi_t && (k >= lo_t || k < sk_t) ? sr[k] : 0xFF800000u;
      }
      float mxs[4] = {__uint_as_float(sr[0]), __uint_as_float(sr[1]), __uint_as_float(sr[2]), __uint_as_float(sr[3])};
#pragma unroll
      for (int j = 4; j + 8 <= 64; j += 8)
#pragma unroll
        for (int k = 0; k < 4; ++k) mxs[k] = ptx::max3(mxs[k], __uint_as_float(sr[j + 2 * k]), __uint_as_float(sr[j + 2 * k + 1]));
#pragma unroll
      for (int k = 0; k < 4; ++k) mxs[k] = fmaxf(mxs[k], __uint_as_float(sr[60 + k]));
      const float mx = fmaxf(fmaxf(mxs[0], mxs[1]), fmaxf(mxs[2], mxs[3])) * qa;
      if (ptx::bar_red_or(bar, 128, !ok || mx > mx_run + kGrow)) {
        s.xch[part][h] = mx;
        if (ptx::bar_red_or(bar, 128, s.abort_flag != 0)) return;  // uniform among the four warps, whoever raised the flag
        const float mxp = fmaxf(fmaxf(s.xch[0][h], s.xch[1][h]), fmaxf(s.xch[2][h], s.xch[3][h]));
        const bool need = mxp > mx_run + kGrow;
        const float mn = need ? mxp : mx_run;
        const float corr = need ? (mx_run == -INFINITY ? 0.f : ptx::ex2(mx_run - mn)) : 1.f;
        l *= corr, mx_run = mn;
        if (t > t0) {  // O holds the item's earlier tiles: wait for their products, then scale this thread's quarter of the row
          const bool okv = ptx::mbar_wait(&s.pv_done, (g - 1) & 1, &s.abort_flag);
          if (ptx::bar_red_or(bar, 128, !okv)) return;
          ptx::tc_fence_after_sync();
#pragma unroll 1
          for (int c0 = 0; c0 < 128; c0 += 32) {
            uint32_t o[32];
            ptx::tmem_ld32(tm_lane + ExtCols::O + 128 * half + c0, o);
            ptx::tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
            ptx::tmem_st32(tm_lane + ExtCols::O + 128 * half + c0, o);
          }
          ptx::tmem_wait_st();
        }
      }
      // P = 2^(s qa - m) as FP16, 64 tokens of the row = 128 bytes
      const float neg_m = mx_run == -INFINITY ? 0.f : -mx_run;
      float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      auto eight = [&](int c, uint32_t (&pk)[4]) {  // weights of tokens 8 c ..
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 x = ptx::fma_f32x2(make_float2(__uint_as_float(sr[8 * c + 2 * k]), __uint_as_float(sr[8 * c + 2 * k + 1])), make_float2(qa, qa),
                                          make_float2(neg_m, neg_m));
          const float2 e = make_float2(ptx::ex2(x.x), ptx::ex2(x.y));
          ls[k & 1] = ptx::add_f32x2(ls[k & 1], e);
          pk[k] = ptx::f32x2_to_f16x2(e.x, e.y);
        }
      };
      constexpr int kHeld = 4;  // sixteen-byte chunks that are ready before the products of the tile before have released P
      uint32_t pk[kHeld > 0 ? kHeld : 1][4];
#pragma unroll
      for (int c = 0; c < kHeld; ++c) eight(c, pk[c]);
      if (g >= 1) ptx::mbar_wait(&s.pv_done, (g - 1) & 1, &s.abort_flag);  // (one that gives up raises the flag; the next vote ends the role)
#pragma unroll
      for (int c = 0; c < kHeld; ++c) ptx::sts128(p_row + (uint32_t(c ^ (h & 7)) << 4), pk[c][0], pk[c][1], pk[c][2], pk[c][3]);
#pragma unroll
      for (int c = kHeld; c < 8; ++c) {
        uint32_t w[4];
        eight(c, w);
        ptx::sts128(p_row + (uint32_t(c ^ (h & 7)) << 4), w[0], w[1], w[2], w[3]);
      }
      l += (ls[0].x + ls[0].y) + (ls[1].x + ls[1].y);
      ptx::fence_proxy_async_smem();
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cta(p_full);
    }

    // ---- end of the item, or of this pair's part of it
    const bool ok = ptx::mbar_wait(&s.pv_done, (g - 1) & 1, &s.abort_flag);
    s.xl[part][h] = l;
    if (ptx::bar_red_or(bar, 128, !ok)) return;
    ptx::tc_fence_after_sync();
    const float lt = (s.xl[0][h] + s.xl[1][h]) + (s.xl[2][h] + s.xl[3][h]);
    const float inv = lt != 0.f ? P.ckv_scale / lt : 0.f;
    const bool whole = t0 == 0 && t1 == m.ntiles;
    // A thread holds a row, but a store of a row per lane touches 32 lines: 128 bytes of 32 rows at a time turn through this warp's
    // 4 KB of s.p (the products that read it are done), so that a store writes four rows' 128 bytes.
    const uint32_t stage = ptx::smem_u32(s.p[0]) + warp * 4096;
    const int c_first = 256 * half + 128 * (quad >> 1);
    const int r_first = 64 * int(rank) + 32 * (quad & 1);  // row of the item in lane 0
    if (whole) {
      uint16_t* const out = P.out + ((long long)m.row0 + r_first) * CKV + c_first;
#pragma unroll 1
      for (int c0 = 0; c0 < 128; c0 += 64) {
        uint32_t v[32];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t o[32];
          ptx::tmem_ld32(tm_lane + ExtCols::O + 128 * half + c0 + 32 * k, o);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) v[16 * k + j] = pack_bf16x2(__uint_as_float(o[2 * j]) * inv, __uint_as_float(o[2 * j + 1]) * inv);
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) ptx::sts128(stage + lane * 128 + (uint32_t(c ^ (lane & 7)) << 4), v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rr = 4 * i + (lane >> 3);
          const uint4 w = ptx::lds128(stage + rr * 128 + (uint32_t((lane ^ rr) & 7) << 4));
          if (r_first + rr < m.rows) *reinterpret_cast<uint4*>(out + rr * CKV + c0 + 8 * (lane & 7)) = w;
        }
        __syncwarp();
      }
    } else {
      const long long slot = 2 * pair + (t0 == 0);
      float* const out = P.o_part + (slot * kExtRows + r_first) * CKV + c_first;
#pragma unroll 1
      for (int c0 = 0; c0 < 128; c0 += 32) {
        uint32_t o[32];
        ptx::tmem_ld32(tm_lane + ExtCols::O + 128 * half + c0, o);
        ptx::tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * inv);
#pragma unroll
        for (int c = 0; c < 8; ++c) ptx::sts128(stage + lane * 128 + (uint32_t(c ^ (lane & 7)) << 4), o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rr = 4 * i + (lane >> 3);
          const uint4 w = ptx::lds128(stage + rr * 128 + (uint32_t((lane ^ rr) & 7) << 4));
          *reinterpret_cast<uint4*>(out + rr * CKV + c0 + 4 * (lane & 7)) = w;
        }
        __syncwarp();
      }
      if (part == 0) P.lse_part[slot * kExtRows + r] = lt != 0.f ? mx_run + log2f(lt) : -INFINITY;
    }
    ptx::tc_fence_before_sync();
    // (also: s.xl, s.xch and the staging rows are used by the next item)
    if (ptx::bar_red_or(bar, 128, s.abort_flag != 0)) return;
    if (lane == 0) ptx::mbar_arrive_cta(o_free);
  }
}

__global__ void __launch_bounds__(kExtThreads, 1)
mla_extend_kernel(const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ CUtensorMap q_map, const ExtParams P) {
  extern __shared__ uint8_t smem_raw[];
  ExtSmem& s = *reinterpret_cast<ExtSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, pair = blockIdx.x >> 1;
  const uint32_t rank = ptx::cluster_ctarank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kExtUnits; ++i) ptx::mbar_init(&s.full[i], 1), ptx::mbar_init(&s.empty[i], 1);
    ptx::mbar_init(&s.q_full, 1), ptx::mbar_init(&s.q_empty, 1);
    for (int i = 0; i < 2; ++i) ptx::mbar_init(&s.s_full[i], 1), ptx::mbar_init(&s.s_free[i], 16);
    ptx::mbar_init(&s.p_full, 16), ptx::mbar_init(&s.pv_done, 1), ptx::mbar_init(&s.o_free, 16);
    s.abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::prefetch_tensormap(&kv_map), ptx::prefetch_tensormap(&q_map);
  }
  if (warp == 10) {
    ptx::tmem_alloc_pair(&s.tmem_base, 512);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::cluster_sync();  // the peer's barriers are initialised too
  ptx::tc_fence_after_sync();
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  if (warp < 8) {
    ext_softmax_role(s, P, pair, rank);
  } else if (warp == 8) {
    if (ptx::elect_one()) ext_producer_role(s, P, &kv_map, &q_map, pair, rank);
  } else if (warp == 9 && rank == 0) {
    if (ptx::elect_one()) ext_mma_role(s, P, pair);
  }
  __syncwarp();
  ptx::tc_fence_before_sync();
  __syncthreads();
  // after a wait that gave up, loads that were issued have landed by the time both CTAs have met
  if (s.abort_flag)
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  ptx::cluster_sync();
  if (warp == 10) ptx::tmem_dealloc_pair(s.tmem_base, 512);
  if (threadIdx.x == 0 && s.abort_flag && P.status) atomicExch(P.status, int(kWaitTimeout));
}

}  // namespace mla
