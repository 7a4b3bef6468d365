// Cache writer: quantise new latent-KV rows to NVFP4 / E4M3 and append them to the paged cache.
//
//   per 16 latent channels: sf = e4m3_rn(amax / 6 / ckv_scale) (saturating at 448), stored as the block scale;
//   code = nearest E2M1 (ties to the even mantissa, magnitudes above 6 saturate) of x / (float(sf) * ckv_scale),
//   0 where the scale is 0; two codes per byte, low nibble = even channel;
//   rope: e4m3_rn(kpe / kpe_scale), saturating.
// Every step is defined as one fp32 IEEE operation in that order, so the bytes are reproducible on a CPU bit for bit.
// The 512 divisions per token would make the kernel instruction-bound, so nothing is divided that a product can settle:
// with the reciprocal of the divisor shrunk and grown by 2^-21, x * r_down and x * r_up enclose the correctly rounded
// quotient (each product is within 5 * 2^-24 of its ideal value), and the result is a monotone step function of the
// magnitude, so if both products round to the same code, the quotient does too. A value that sits closer to a rounding
// boundary is settled on its own: a latent value that ties exactly (BF16 inputs do in a few percent of the scale blocks) by
// one fused multiply-add, anything else by the real division. The block scale and the rope pair are treated alike; a
// power-of-two rope scale needs no enclosure, its products are exact.
//
// 1152 bytes in, 352 bytes out per token, bound by instruction issue (343 warp instructions per token, 73 % of the issue slots):
// 596415 tokens in 219.6 us, 233.7 with the divisions of the block scale and the rope (138 at the measured copy bandwidth).
// Thirty-two tokens per warp with one walk through the page tables for all of them was slower (246.7 us).
// One warp per token per trip; lane l owns scale block l
// (channels 16l .. 16l+15: two 16-byte loads, one 8-byte store, the warp writes the token's 256 packed bytes as one
// contiguous run) and rope channels 2l, 2l+1.
#pragma once
#include <cuda_bf16.h>
#include "mla_common.cuh"
#include "mla_dequant.cuh"  // e4m3_value

namespace mla {

constexpr int kQuantThreads = 256;

__device__ __forceinline__ uint32_t f32x2_to_e4m3x2_sat(float lo, float hi) {  // lo -> low byte
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
// eight floats -> eight E2M1 codes (round to nearest even, saturating), value 0 in the lowest nibble
__device__ __forceinline__ uint32_t e2m1x8(const float (&y)[8]) {
  uint32_t d;
  asm("{\n.reg .b8 b0, b1, b2, b3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      "mov.b32 %0, {b0, b1, b2, b3};\n}"
      : "=r"(d)
      : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  return d;
}
__device__ __forceinline__ uint32_t e2m1_code(float y) {
  // thresholds halfway between 0, .5, 1, 1.5, 2, 3, 4, 6; a tie goes to the code with the even mantissa bit
  const float a = fabsf(y);
  const uint32_t mag = uint32_t(a > 0.25f) + uint32_t(a >= 0.75f) + uint32_t(a > 1.25f) + uint32_t(a >= 1.75f) +
                       uint32_t(a > 2.5f) + uint32_t(a >= 3.5f) + uint32_t(a > 5.0f);
  return mag | ((__float_as_uint(y) >> 28) & 8u);
}

// Reciprocals of the divisors that are the same for every token, as enclosures; divisors near the ends of the fp32 range
// (where a product or a reciprocal need not be a normal number) take the divisions.
constexpr float kQuantDown = 1.f - 0x1p-21f, kQuantUp = 1.f + 0x1p-21f;
struct QuantScales {
  float ckv_scale, kpe_scale, six_dn, six_up, kpe_dn, kpe_up;
  bool fast_sf, fast_kpe;
  __device__ __forceinline__ QuantScales(float ckv, float kpe) : ckv_scale(ckv), kpe_scale(kpe) {
    auto ordinary = [](float d) { return d > 0x1p-100f && d < 0x1p100f; };
    const float six = __fmul_rn(6.0f, ckv), r_six = __frcp_rn(six), r_kpe = __frcp_rn(kpe);
    fast_sf = ordinary(six), fast_kpe = ordinary(kpe);
    const bool kpe_pow2 = (__float_as_uint(kpe) & 0x007FFFFFu) == 0u;
    six_dn = r_six * kQuantDown, six_up = r_six * kQuantUp;
    kpe_dn = kpe_pow2 ? r_kpe : r_kpe * kQuantDown, kpe_up = kpe_pow2 ? r_kpe : r_kpe * kQuantUp;
  }
};

// Codes and scale byte of one block of 16 latent values; `value(j)` gives value j again.
struct QuantBlock {
  uint32_t lo, hi, sf8;
};
template <class Value>
__device__ __forceinline__ QuantBlock quantize_block(const float (&x)[16], const QuantScales& Q, Value value) {
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fmaxf(fabsf(x[2 * j]), fabsf(x[2 * j + 1])));
  const uint32_t sf2 = f32x2_to_e4m3x2_sat(amax * Q.six_dn, amax * Q.six_up);
  uint32_t sf8 = sf2 & 0xFFu;
  if (!Q.fast_sf || sf8 != sf2 >> 8) sf8 = f32x2_to_e4m3x2_sat(__fdiv_rn(__fdiv_rn(amax, 6.0f), Q.ckv_scale), 0.f) & 0xFFu;
  const float sf = __fmul_rn(e4m3_value(uint8_t(sf8)), Q.ckv_scale);
  uint32_t lo = 0, hi = 0;
  if (sf > 0.f) {
    const float r = __frcp_rn(sf), rd = r * kQuantDown, ru = r * kQuantUp;
    float yd[16], yu[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) yd[j] = x[j] * rd, yu[j] = x[j] * ru;
    lo = e2m1x8(reinterpret_cast<const float(&)[8]>(yd[0])), hi = e2m1x8(reinterpret_cast<const float(&)[8]>(yd[8]));
    const uint32_t dlo = lo ^ e2m1x8(reinterpret_cast<const float(&)[8]>(yu[0]));
    const uint32_t dhi = hi ^ e2m1x8(reinterpret_cast<const float(&)[8]>(yu[8]));
    // Some values are within 2^-21 of a rounding boundary: for those the defining computation decides. Nearly all of
    // them are exact ties (BF16 inputs over a scale of a few bits): every boundary has at most three significant
    // bits, so the candidate T is the product rounded to three bits, and T * sf == |x| (one fused multiply-add,
    // exact in sign and in zero) proves that x / sf is T itself; only the rest take the division. The loop visits
    // the flagged values alone.
    auto settle = [&](uint32_t codes, uint32_t diff, int base) {
      while (diff) {
        const int j = (__ffs(diff) - 1) >> 2;
        diff &= ~(15u << (4 * j));
        const float xv = value(base + j);
        const float tie = __uint_as_float((__float_as_uint(fabsf(xv) * r) + 0x00100000u) & 0xFFE00000u);
        const float q = __fmaf_rn(tie, sf, -fabsf(xv)) == 0.f ? copysignf(tie, xv) : __fdiv_rn(xv, sf);
        codes = (codes & ~(15u << (4 * j))) | (e2m1_code(q) << (4 * j));
      }
      return codes;
    };
    lo = settle(lo, dlo, 0), hi = settle(hi, dhi, 8);
  }
  return {lo, hi, sf8};
}

// e4m3(x0 / kpe_scale) in the low byte, e4m3(x1 / kpe_scale) in the next
__device__ __forceinline__ uint32_t quantize_rope_pair(float x0, float x1, const QuantScales& Q) {
  uint32_t k8 = f32x2_to_e4m3x2_sat(x0 * Q.kpe_dn, x1 * Q.kpe_dn);
  if (!Q.fast_kpe || k8 != f32x2_to_e4m3x2_sat(x0 * Q.kpe_up, x1 * Q.kpe_up))
    k8 = f32x2_to_e4m3x2_sat(__fdiv_rn(x0, Q.kpe_scale), __fdiv_rn(x1, Q.kpe_scale));
  return k8;
}

// cache row of position `pos` of request `b`; negative if the request, the position or the page lies outside the tables
__device__ __forceinline__ long long cache_row(int b, int pos, long long num_pages, int page_shift, const int* kv_indices,
                                               const int* kv_indptr, int batch) {
  if (b < 0 || b >= batch || pos < 0) return -1;
  const int first = kv_indptr[b], npages = kv_indptr[b + 1] - first, pi = pos >> page_shift;
  if (pi >= npages) return -1;
  const int page = kv_indices[first + pi];
  if (page < 0 || page >= num_pages) return -1;
  return ((long long)page << page_shift) + (pos & ((1 << page_shift) - 1));
}

// status: optional device word, set to 1 if a token named a request, position or page outside the tables (the token
// is skipped, nothing is written for it).
__global__ void __launch_bounds__(kQuantThreads)
mla_quantize_append_kernel(const __nv_bfloat16* __restrict__ ckv, const __nv_bfloat16* __restrict__ kpe,
                           const int* __restrict__ batch_indices, const int* __restrict__ positions, long long nnz,
                           uint8_t* __restrict__ ckv_cache, uint8_t* __restrict__ sf_cache, uint8_t* __restrict__ kpe_cache,
                           long long num_pages, int page_shift, const int* __restrict__ kv_indices,
                           const int* __restrict__ kv_indptr, int batch, float ckv_scale, float kpe_scale, int* status) {
  const int lane = threadIdx.x & 31;
  const QuantScales Q(ckv_scale, kpe_scale);
  const long long warp0 = (long long)blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);
  const long long stride = (long long)gridDim.x * (kQuantThreads / 32);
  for (long long t = warp0; t < nnz; t += stride) {
    // the row itself does not wait for the walk through the page tables
    const uint4* src = reinterpret_cast<const uint4*>(ckv + t * CKV + 16 * lane);
    const uint4 w0 = src[0], w1 = src[1];
    const uint32_t rope = reinterpret_cast<const uint32_t*>(kpe + t * KPE)[lane];
    const int b = batch_indices[t], pos = positions[t];
    const long long row = cache_row(b, pos, num_pages, page_shift, kv_indices, kv_indptr, batch);
    if (row < 0) {
      if (lane == 0 && status) *status = 1;
      continue;
    }
    // ---- latent block `lane`
    const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
    float x[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[2 * j] = __uint_as_float(w[j] << 16), x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    // (a value that has to be settled is read again from memory: the registers cannot be indexed)
    const QuantBlock q = quantize_block(x, Q, [&](int j) { return __bfloat162float(ckv[t * CKV + 16 * lane + j]); });
    *reinterpret_cast<uint2*>(ckv_cache + row * (CKV / 2) + 8 * lane) = make_uint2(q.lo, q.hi);
    sf_cache[row * (CKV / 16) + lane] = uint8_t(q.sf8);
    // ---- rope channels 2 lane, 2 lane + 1
    reinterpret_cast<uint16_t*>(kpe_cache + row * KPE)[lane] =
        uint16_t(quantize_rope_pair(__uint_as_float(rope << 16), __uint_as_float(rope & 0xFFFF0000u), Q));
  }
}

// ---------------------------------------------------------------------------------------------------------------
// The writer behind the latent projection: its raw rows [latent 512 | rope 64] are normalised, rotated, quantised and appended in
// one pass.
//
//   latent : y_c = w_c x_c / sqrt(mean(x^2) + eps), as an fp32 number (correctly rounded), then as BF16
//   rope   : the pair (a, b) of position p turns into (a cos - b sin, b cos + a sin) with row p of the cos | sin table, as an
//            fp32 number, then as BF16
//   then the writer's own steps (above): the bytes are those of mla_quantize_append_kernel on the BF16 rows.
// A code of the cache changes by a whole step where a value crosses a rounding border, so the BF16 values themselves are exact:
// the sum of squares is taken in 64 bits, the product with the reciprocal root in fp32 (within two units in the last place of
// the defined one), and a product that close to a BF16 border (one in ten thousand) again in 64 bits. The rope products are taken in
// 64 bits at once: they cancel, and there are two per lane.
//
// One warp per token per trip, lane l = scale block l, as above; a lane's normalised BF16 values sit in shared memory for the few that
// have to be settled.
// ---------------------------------------------------------------------------------------------------------------
template <bool INTERLEAVED>
__global__ void __launch_bounds__(kQuantThreads)
mla_norm_rope_append_kernel(const __nv_bfloat16* __restrict__ ckv, long long ckv_stride, const __nv_bfloat16* __restrict__ kpe,
                            long long kpe_stride, const __nv_bfloat16* __restrict__ weight, const float* __restrict__ cos_sin,
                            int max_pos, double eps, const int* __restrict__ batch_indices, const int* __restrict__ positions,
                            long long nnz, uint8_t* __restrict__ ckv_cache, uint8_t* __restrict__ sf_cache,
                            uint8_t* __restrict__ kpe_cache, long long num_pages, int page_shift,
                            const int* __restrict__ kv_indices, const int* __restrict__ kv_indptr, int batch, float ckv_scale,
                            float kpe_scale, int* status) {
  __shared__ uint32_t held[kQuantThreads][9];  // a lane's 16 values, rows of nine words: no bank conflicts
  const int lane = threadIdx.x & 31;
  const QuantScales Q(ckv_scale, kpe_scale);
  uint32_t wt[8];
  {
    const uint4* src = reinterpret_cast<const uint4*>(weight + 16 * lane);
    const uint4 a = __ldg(src), b = __ldg(src + 1);
    wt[0] = a.x, wt[1] = a.y, wt[2] = a.z, wt[3] = a.w, wt[4] = b.x, wt[5] = b.y, wt[6] = b.z, wt[7] = b.w;
  }
  const long long warp0 = (long long)blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);
  const long long stride = (long long)gridDim.x * (kQuantThreads / 32);
  for (long long t = warp0; t < nnz; t += stride) {
    const uint4* src = reinterpret_cast<const uint4*>(ckv + t * ckv_stride + 16 * lane);
    const uint4 w0 = src[0], w1 = src[1];
    const __nv_bfloat16* rp = kpe + t * kpe_stride;
    float a, b;
    if constexpr (INTERLEAVED) {
      const uint32_t rope = reinterpret_cast<const uint32_t*>(rp)[lane];
      a = __uint_as_float(rope << 16), b = __uint_as_float(rope & 0xFFFF0000u);
    } else {
      a = __bfloat162float(rp[lane]), b = __bfloat162float(rp[32 + lane]);
    }
    const int pos = positions[t];
    const long long row = pos < max_pos ? cache_row(batch_indices[t], pos, num_pages, page_shift, kv_indices, kv_indptr, batch) : -1;
    if (row < 0) {
      if (lane == 0 && status) *status = 1;
      continue;
    }
    const float cs = __ldg(cos_sin + (long long)pos * KPE + lane), sn = __ldg(cos_sin + (long long)pos * KPE + 32 + lane);
    const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
    double sum = 0.;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double u = double(__uint_as_float(w[j] << 16)), v = double(__uint_as_float(w[j] & 0xFFFF0000u));
      sum = fma(u, u, sum), sum = fma(v, v, sum);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    const double r = rsqrt(sum * (1. / CKV) + eps);
    const float rf = float(r);
    const bool plain_row = rf > 0x1p-60f && rf < 0x1p60f;
    float x[16];
    uint32_t* const mine = held[threadIdx.x];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t pair = 0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float xv = __uint_as_float(e ? w[j] & 0xFFFF0000u : w[j] << 16), wv = __uint_as_float(e ? wt[j] & 0xFFFF0000u : wt[j] << 16);
        const float p = __fmul_rn(xv, wv);  // exact: eight bits times eight bits
        float y = __fmul_rn(p, rf);
        const uint32_t low = (__float_as_uint(y) - 0x7FFDu) & 0xFFFFu;  // up to 6: within three units of a BF16 border
        const float size = fabsf(p);
        if (low <= 6u || !plain_row || !(size > 0x1p-60f && size < 0x1p60f)) y = float(double(xv) * double(wv) * r);
        const uint32_t h = __bfloat16_as_ushort(__float2bfloat16_rn(y));
        x[2 * j + e] = __uint_as_float(h << 16);
        pair |= h << (16 * e);
      }
      mine[j] = pair;
    }
    const QuantBlock q = quantize_block(x, Q, [&](int j) { return __uint_as_float(j & 1 ? mine[j >> 1] & 0xFFFF0000u : mine[j >> 1] << 16); });
    *reinterpret_cast<uint2*>(ckv_cache + row * (CKV / 2) + 8 * lane) = make_uint2(q.lo, q.hi);
    sf_cache[row * (CKV / 16) + lane] = uint8_t(q.sf8);
    const double c = double(cs), s = double(sn);
    const float x0 = __bfloat162float(__float2bfloat16_rn(float(fma(double(a), c, -(double(b) * s)))));
    const float x1 = __bfloat162float(__float2bfloat16_rn(float(fma(double(b), c, double(a) * s))));
    const uint32_t k8 = quantize_rope_pair(x0, x1, Q);
    if constexpr (INTERLEAVED) {
      reinterpret_cast<uint16_t*>(kpe_cache + row * KPE)[lane] = uint16_t(k8);
    } else {
      kpe_cache[row * KPE + lane] = uint8_t(k8), kpe_cache[row * KPE + 32 + lane] = uint8_t(k8 >> 8);
    }
  }
}

}  // namespace mla
