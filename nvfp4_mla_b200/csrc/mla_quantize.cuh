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
// 1152 bytes in, 352 bytes out per token, bound by instruction issue (1 048 576 tokens with a power of two as ckv_scale: 327 warp instructions
// per token, 77 % of the issue slots): 596 415 tokens in 195 us (137 at the measured copy bandwidth), 220 with one instruction per product
// instead of two products per instruction and 64-bit rows; 275 015 tokens 96 us, 114 with a power of two, where more values tie. Thirty-two
// tokens per warp with one walk through the page tables for all of them was slower (246.7 us for the 596 415).
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

// A factor f for the block scale `sf8` with which every BF16 value x has code(fl(x f)) = code(fl(x / sf)); where there is none, the
// reciprocal f, rounded down, and a second term g >= 0 with which fl(x f + fl(x g)) has the code; {0, 0} if that is none either. (With g < 0
// the two products of x = -0 would have opposite signs and their sum would be +0, another code than -0 / sf.)
// Both quotients round alike unless x / sf is within 2^-20 of a boundary; a boundary is m 2^k with m = 1, 1.25, 1.5 or 1.75, so only the
// BF16 number x_m next to m sf can be that close (and its products with powers of two, which behave like it), and the scale alone
// says whether it is: fl(m sf) is then within 16 units in its last place of a BF16 number. For these m (none for most scales, one or
// two for amax / (6 * 448) of a BF16 amax, all four where the cache's scale is a power of two) f has to put x_m on the side of m,
// or on m itself, that the division does; f is the reciprocal or one of the two numbers on either side of it, within 3 * 2^-23 of 1 / sf.
__device__ __forceinline__ float2 quant_factor(uint32_t sf8, float ckv_scale) {
  const float sf = __fmul_rn(e4m3_value(uint8_t(sf8)), ckv_scale);
  if (!(sf > 0x1p-100f && sf < 0x1p100f)) return make_float2(0.f, 0.f);
  const uint32_t r = __float_as_uint(__frcp_rn(sf));
  float x[4];   // x_m, or m itself over ...
  float q[4];   // ... and its quotient
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t t = __float_as_uint(__fmul_rn(sf, 1.f + 0.25f * i)) + 16u;
    x[i] = (t & 0xFFFFu) <= 32u ? __uint_as_float(t & 0xFFFF0000u) : 0.f;
    q[i] = __fdiv_rn(x[i], sf);
  }
#pragma unroll
  for (int j = 0; j < 5; ++j) {
    const float f = __uint_as_float(r + (j & 1 ? -((j + 1) >> 1) : j >> 1));
    bool good = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float m = 1.f + 0.25f * i, p = __fmul_rn(x[i], f);
      good &= (p < m) == (q[i] < m) && (p > m) == (q[i] > m);
    }
    if (good) return make_float2(f, 0.f);
  }
  const float f = __uint_as_float(__fmaf_rn(-sf, __uint_as_float(r), 1.f) < 0.f ? r - 1 : r), g = __fmul_rn(__fmaf_rn(-sf, f, 1.f), f);
  bool good = sf8 != 0x7Eu;  // (the largest scale's block may hold infinities)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float m = 1.f + 0.25f * i, p = __fmaf_rn(x[i], f, __fmul_rn(x[i], g));
    good &= (p < m) == (q[i] < m) && (p > m) == (q[i] > m);
  }
  return good ? make_float2(f, g) : make_float2(0.f, 0.f);
}
constexpr int kQuantFactors = 128;
struct QuantFactors {
  float f[kQuantFactors], g[kQuantFactors];
};
// by the block, synchronises; whether some block scale needs its second term (then all products take both, 0 for the others)
__device__ __forceinline__ bool quant_factors(QuantFactors& s, float ckv_scale) {  // by the block; synchronises
  const bool mine = threadIdx.x < kQuantFactors;
  const float2 f = mine ? quant_factor(threadIdx.x, ckv_scale) : make_float2(0.f, 0.f);
  const bool second = __syncthreads_or(f.y != 0.f);
  // (0 * inf: where second terms are taken, a block that may hold infinities has no factor)
  if (mine) s.f[threadIdx.x] = second && threadIdx.x == 0x7Eu ? 0.f : f.x, s.g[threadIdx.x] = f.y;
  __syncthreads();
  return second;
}

// Codes and scale byte of one block of 16 latent values; `value(j)` gives value j again. With FACTORS one product per value settles its code.
struct QuantBlock {
  uint32_t lo, hi, sf8;
};
template <bool FACTORS, class Value>
__device__ __forceinline__ QuantBlock quantize_block(const float (&x)[16], const QuantScales& Q, const QuantFactors* factors, bool second, Value value) {
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) amax = ptx::max3(amax, fabsf(x[2 * j]), fabsf(x[2 * j + 1]));
  const uint32_t sf2 = f32x2_to_e4m3x2_sat(amax * Q.six_dn, amax * Q.six_up);
  uint32_t sf8 = sf2 & 0xFFu;
  if (!Q.fast_sf || sf8 != sf2 >> 8) sf8 = f32x2_to_e4m3x2_sat(__fdiv_rn(__fdiv_rn(amax, 6.0f), Q.ckv_scale), 0.f) & 0xFFu;
  if constexpr (FACTORS) {
    const float f = factors->f[sf8 & 127u];
    if (f != 0.f) {
      float y[16];
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        const float2 p = ptx::mul_f32x2(make_float2(x[j], x[j + 1]), make_float2(f, f));
        y[j] = p.x, y[j + 1] = p.y;
      }
      if (second) {
        const float g = factors->g[sf8 & 127u];
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const float2 v = make_float2(x[j], x[j + 1]), p = ptx::fma_f32x2(v, make_float2(f, f), ptx::mul_f32x2(v, make_float2(g, g)));
          y[j] = p.x, y[j + 1] = p.y;
        }
      }
      return {e2m1x8(reinterpret_cast<const float(&)[8]>(y[0])), e2m1x8(reinterpret_cast<const float(&)[8]>(y[8])), sf8};
    }
  }
  const float sf = __fmul_rn(e4m3_value(uint8_t(sf8)), Q.ckv_scale);
  uint32_t lo = 0, hi = 0;
  if (sf > 0.f) {
    const float r = __frcp_rn(sf);
    const float rd = r * kQuantDown, ru = r * kQuantUp;
    float yd[16], yu[16];
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      const float2 d = ptx::mul_f32x2(make_float2(x[j], x[j + 1]), make_float2(rd, rd)), u = ptx::mul_f32x2(make_float2(x[j], x[j + 1]), make_float2(ru, ru));
      yd[j] = d.x, yd[j + 1] = d.y, yu[j] = u.x, yu[j + 1] = u.y;
    }
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
__device__ __forceinline__ int cache_row(int b, int pos, int num_pages, int page_shift, const int* kv_indices, const int* kv_indptr, int batch) {
  if (b < 0 || b >= batch || pos < 0) return -1;
  const int first = kv_indptr[b], npages = kv_indptr[b + 1] - first, pi = pos >> page_shift;
  if (pi >= npages) return -1;
  const int page = kv_indices[first + pi];
  if (page < 0 || page >= num_pages) return -1;
  return (page << page_shift) + (pos & ((1 << page_shift) - 1));  // (the pool has fewer than 2^31 rows)
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
    const long long row = cache_row(b, pos, int(num_pages), page_shift, kv_indices, kv_indptr, batch);
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
    const QuantBlock q = quantize_block<false>(x, Q, nullptr, false, [&](int j) { return __bfloat162float(ckv[t * CKV + 16 * lane + j]); });
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
// A code of the cache changes by a whole step where a value crosses a rounding border, so the BF16 values themselves are exact. They
// are computed in fp32 with an error bound, and a value that close to a BF16 border is computed again in 64 bits:
//   latent: the squares are exact in fp32 (eight bits times eight), their sum passes ten rounding additions (five in a lane, five
//           shuffles): within 10 * 2^-24 of itself; eps and its addition (2 * 2^-24 of the mean, half of it in the root),
//           the reciprocal root (two units) and the product (x w is exact) make y off by at most 11 units in its last place. One
//           value in 2600 is that close to a border, one token in five has such a value.
//   rope  : a cos - b sin as fma(a, cos, -p) - fma(b, sin, -p) with p = b sin rounded, which is within two units of the defined number.
//
// One warp per token per trip, lane l = scale block l, as above; a lane's normalised BF16 values sit in shared memory for the few that
// have to be settled, the weights and the factors of the 128 block scales there too. A lane looks up the place of one of the warp's next
// 32 tokens, so that the walk through the page tables is paid for once in 32 trips. 1512 bytes per token, bound by instruction issue and
// the latency of a warp's chain of steps (347 warp instructions per token, 67 % of the issue slots): 275 015 tokens in 134 us with
// ckv_scale = 6.5 / (6 * 448) (63 at the measured copy bandwidth), 143 with a power of two, where a third of the block scales needs a
// second term (172 with the enclosing products for these, the two here at 128 and 137 on that box). Before: 166 and 188 with the enclosing products of the writer above and a walk per token; 345 with the norm in 64 bits
// throughout. Rows fetched ahead into shared memory (134), 40 warps per SM (171) and two CTAs per resident one (129.5) gained nothing.
// ---------------------------------------------------------------------------------------------------------------
template <bool INTERLEAVED>
__global__ void __launch_bounds__(kQuantThreads, 4)
mla_norm_rope_append_kernel(const __nv_bfloat16* __restrict__ ckv, long long ckv_stride, const __nv_bfloat16* __restrict__ kpe,
                            long long kpe_stride, const __nv_bfloat16* __restrict__ weight, const float* __restrict__ cos_sin,
                            int max_pos, double eps, const int* __restrict__ batch_indices, const int* __restrict__ positions,
                            long long nnz, uint8_t* __restrict__ ckv_cache, uint8_t* __restrict__ sf_cache,
                            uint8_t* __restrict__ kpe_cache, long long num_pages, int page_shift,
                            const int* __restrict__ kv_indices, const int* __restrict__ kv_indptr, int batch, float ckv_scale,
                            float kpe_scale, int* status) {
  __shared__ uint4 held[2][kQuantThreads];  // a lane's 16 normalised values
  __shared__ float4 gains[4][32];           // the weights: lane l's 16
  __shared__ QuantFactors factors;
  const int lane = threadIdx.x & 31;
  const QuantScales Q(ckv_scale, kpe_scale);
  const float eps_f = float(eps);
  // Weights: 0 or of ordinary size. A product below fp32's normal numbers (not exact) then stands for a y below 2^-96, whose code is 0
  // whatever its error, unless the cache's scale is that small as well.
  bool ordinary_gains = ckv_scale > 0x1p-80f;
  for (int i = threadIdx.x; i < CKV; i += kQuantThreads) {
    const float g = __bfloat162float(weight[i]);
    reinterpret_cast<float*>(&gains[(i & 15) >> 2][i >> 4])[i & 3] = g;
    ordinary_gains &= g == 0.f || (fabsf(g) > 0x1p-20f && fabsf(g) < 0x1p20f);
  }
  const bool second = quant_factors(factors, ckv_scale);
  ordinary_gains = __syncthreads_and(ordinary_gains);
  const long long warp0 = (long long)blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);
  const long long stride = (long long)gridDim.x * (kQuantThreads / 32);
  // A lane looks up the place of one of the warp's next 32 tokens: one walk through the page tables for all of them.
  int places = -1, at = 0;
  int trip = 0;
  for (long long t = warp0; t < nnz; t += stride, ++trip) {
    if ((trip & 31) == 0) {
      const long long mine = t + lane * stride;
      if (mine < nnz) {
        at = positions[mine];
        places = at < max_pos ? cache_row(batch_indices[mine], at, int(num_pages), page_shift, kv_indices, kv_indptr, batch) : -1;
      }
    }
    const uint4* src = reinterpret_cast<const uint4*>(ckv + t * ckv_stride + 16 * lane);
    const uint4 w0 = __ldcs(src), w1 = __ldcs(src + 1);
    const __nv_bfloat16* rp = kpe + t * kpe_stride;
    uint32_t rope;  // interleaved: the pair; else channel `lane` and, above it, channel 32 + lane
    if constexpr (INTERLEAVED) rope = __ldcs(reinterpret_cast<const uint32_t*>(rp) + lane);
    else rope = uint32_t(__ldcs(reinterpret_cast<const uint16_t*>(rp) + lane)) | uint32_t(__ldcs(reinterpret_cast<const uint16_t*>(rp) + 32 + lane)) << 16;
    const float a = __uint_as_float(rope << 16), b = __uint_as_float(rope & 0xFFFF0000u);
    const int pos = __shfl_sync(~0u, at, trip & 31);
    const bool rotated = uint32_t(pos) < uint32_t(max_pos);
    const float cs = rotated ? __ldg(cos_sin + (long long)pos * KPE + lane) : 0.f, sn = rotated ? __ldg(cos_sin + (long long)pos * KPE + 32 + lane) : 0.f;
    const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
    auto two = [](uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)); };
    float2 sq[2];  // two chains of four
#pragma unroll
    for (int j = 0; j < 8; ++j) sq[j & 1] = j < 2 ? ptx::mul_f32x2(two(w[j]), two(w[j])) : ptx::fma_f32x2(two(w[j]), two(w[j]), sq[j & 1]);
    sq[0] = ptx::add_f32x2(sq[0], sq[1]);
    float sum = __fadd_rn(sq[0].x, sq[0].y);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(~0u, sum, o));
    const float mean = __fadd_rn(sum * (1.f / CKV), eps_f), r = rsqrtf(mean);
    // (fp32 holds the row and the products well inside its range)
    const bool ordinary = mean > 0x1p-60f && mean < 0x1p60f && ordinary_gains;
    uint32_t held_[8], nearest = 0xFFFFFFFFu;  // smallest distance to a border seen, two at a time: (low half of y) - 0x8000 + 12
    auto gain4 = [&](int k) { return gains[k][lane]; };  // weights 4k .. of the lane
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 g = gain4(k);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = 2 * k + e;
        const float2 y = ptx::mul_f32x2(ptx::mul_f32x2(two(w[j]), e ? make_float2(g.z, g.w) : make_float2(g.x, g.y)), make_float2(r, r));
        nearest = __viaddmin_u16x2(__byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x5410), 0x800C800Cu, nearest);
        held_[j] = ptx::f32x2_to_bf16x2(y.x, y.y);
      }
    }
    const bool near = (nearest & 0xFFFFu) <= 24u || nearest >> 16 <= 24u || !ordinary;
    if (__any_sync(~0u, near)) {
      double s2 = 0.;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double u = double(two(w[j]).x), v = double(two(w[j]).y);
        s2 = fma(u, u, s2), s2 = fma(v, v, s2);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) s2 += __shfl_xor_sync(~0u, s2, o);
      const double rd = rsqrt(s2 * (1. / CKV) + eps);
      if (near) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 g = gain4(j >> 1);
          const float2 a2 = two(w[j]), g2 = j & 1 ? make_float2(g.z, g.w) : make_float2(g.x, g.y);
          held_[j] = ptx::f32x2_to_bf16x2(float(double(a2.x) * double(g2.x) * rd), float(double(a2.y) * double(g2.y) * rd));
        }
      }
    }
    held[0][threadIdx.x] = make_uint4(held_[0], held_[1], held_[2], held_[3]), held[1][threadIdx.x] = make_uint4(held_[4], held_[5], held_[6], held_[7]);
    float x[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[2 * j] = two(held_[j]).x, x[2 * j + 1] = two(held_[j]).y;
    const QuantBlock q = quantize_block<true>(x, Q, &factors, second, [&](int j) {
      const uint32_t v = reinterpret_cast<const uint32_t*>(&held[j >> 3][threadIdx.x])[j >> 1 & 3];
      return __uint_as_float(j & 1 ? v & 0xFFFF0000u : v << 16);
    });
    const long long row = __shfl_sync(~0u, places, trip & 31);
    if (row < 0) {
      if (lane == 0 && status) *status = 1;
      continue;
    }
    *reinterpret_cast<uint2*>(ckv_cache + row * (CKV / 2) + 8 * lane) = make_uint2(q.lo, q.hi);
    sf_cache[row * (CKV / 16) + lane] = uint8_t(q.sf8);
    const float p0 = __fmul_rn(b, sn), p1 = __fmul_rn(a, sn);
    float x0 = __fsub_rn(__fmaf_rn(a, cs, -p0), __fmaf_rn(b, sn, -p0)), x1 = __fadd_rn(__fmaf_rn(b, cs, p1), __fmaf_rn(a, sn, -p1));
    // (very small: the products' errors may be below fp32's range; very large or NaN: something may have overflowed)
    const bool odd = fminf(fabsf(x0), fabsf(x1)) < 0x1p-60f || !(fabsf(x0) + fabsf(x1) < 0x1p100f);
    const uint32_t border = __viaddmin_u16x2(__byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x5410), 0x80038003u, 0xFFFFFFFFu);
    if ((border & 0xFFFFu) <= 6u || border >> 16 <= 6u || odd) {
      const double da = double(a), db = double(b), dc = double(cs), ds = double(sn);
      x0 = float(fma(da, dc, -(db * ds))), x1 = float(fma(db, dc, da * ds));
    }
    x0 = __bfloat162float(__float2bfloat16_rn(x0)), x1 = __bfloat162float(__float2bfloat16_rn(x1));
    const uint32_t k8 = quantize_rope_pair(x0, x1, Q);
    if constexpr (INTERLEAVED) {
      reinterpret_cast<uint16_t*>(kpe_cache + row * KPE)[lane] = uint16_t(k8);
    } else {
      kpe_cache[row * KPE + lane] = uint8_t(k8), kpe_cache[row * KPE + 32 + lane] = uint8_t(k8 >> 8);
    }
  }
}

}  // namespace mla
