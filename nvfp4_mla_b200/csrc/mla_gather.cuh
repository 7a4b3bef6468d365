// Reading the cache back: ranges of tokens of the requests, out of the pages, dequantised into contiguous rows (the context of a
// prefill step for an up-projection that takes BF16 rows). The arithmetic is that of the whole-cache dequantisation
// (mla_dequant.cuh): e2m1 * block_scale * ckv_scale, each product rounded to fp32, then to the output type.
//
// Output row i belongs to the request b with indptr[b] <= i < indptr[b + 1] and holds its token starts[b] + i - indptr[b].
// HBM-bound: 352 bytes in, 1152 (bf16) or 2304 (fp32) bytes out per row. A warp takes four rows: a lane finds the cache row of each
// (binary search over the indptr, then the page table: a chain of dependent loads that the rows pay once), then all lanes convert
// them two at a time, each instruction of the warp one contiguous run. 530846 rows to BF16: 127 us, 0.96 of the measured copy bandwidth
// (32 rows per warp 142, 8 rows 133, 2 rows 133: long runs leave too few warps in their loads, short ones pay for the look-up).
#pragma once
#include <cuda_bf16.h>
#include "mla_common.cuh"
#include "mla_dequant.cuh"

namespace mla {

constexpr int kGatherThreads = 256;
constexpr int kGatherRows = 4;  // rows of a warp (two trips); two where there are too few to give every SM its warps

// status: optional device word, set to 1 if a row's token lies outside the page table or on a page outside the cache (its output is 0)
template <typename T>
__global__ void __launch_bounds__(kGatherThreads)
mla_gather_kernel(const uint8_t* __restrict__ ckv, const uint8_t* __restrict__ sf, const uint8_t* __restrict__ kpe, long long num_pages,
                  int page_shift, const int* __restrict__ page_table, long long pt_stride, int pt_width, const int* __restrict__ indptr,
                  const int* __restrict__ starts, int batch, int total, int rows_per_warp, float ckv_scale, float kpe_scale,
                  T* __restrict__ ckv_out, T* __restrict__ kpe_out, int* status) {
  constexpr int U = kDequantTokens, L = sizeof(T) == 2 ? 2 : 4;  // L loads of 512 / L channels per token
  const int lane = threadIdx.x & 31;
  const long long warp = (long long)blockIdx.x * (kGatherThreads / 32) + (threadIdx.x >> 5);
  const long long r0 = warp * rows_per_warp;
  const int first = __ldg(indptr), last = __ldg(indptr + batch) < total ? __ldg(indptr + batch) : total;  // rows outside are left as they are
  if (r0 >= last) return;
  const int mine = int(r0) + lane;  // the row this lane looks up
  long long src = -2;               // its cache row, -1: zeros, -2: not a row of this warp
  if (lane < rows_per_warp && mine < last && mine >= first) {
    const int b = request_of_row(indptr, batch, mine);
    const long long tok = (long long)(starts ? __ldg(starts + b) : 0) + (mine - __ldg(indptr + b));
    src = -1;
    if (tok >= 0 && (tok >> page_shift) < pt_width) {
      const int page = __ldg(page_table + (long long)b * pt_stride + (tok >> page_shift));
      if (page >= 0 && page < num_pages) src = ((long long)page << page_shift) + (tok & ((1 << page_shift) - 1));
    }
    if (src < 0 && status) *status = 1;
  }
  for (int i = 0; i < rows_per_warp; i += U) {
    uint32_t w[U][L], sv[U], two[U];
    long long at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      at[u] = __shfl_sync(~0u, src, i + u);
      const long long tok = at[u] < 0 ? 0 : at[u];
      sv[u] = __ldcs(sf + tok * (CKV / 16) + lane);
#pragma unroll
      for (int j = 0; j < L; ++j) {
        if constexpr (L == 2) w[u][j] = __ldcs(reinterpret_cast<const uint32_t*>(ckv + tok * (CKV / 2) + 128 * j) + lane);
        else w[u][j] = __ldcs(reinterpret_cast<const uint16_t*>(ckv + tok * (CKV / 2) + 64 * j) + lane);
      }
      two[u] = __ldcs(reinterpret_cast<const uint16_t*>(kpe + tok * KPE) + lane);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (at[u] == -2) continue;
      if (at[u] < 0) {
        sv[u] = 0, two[u] = 0;
#pragma unroll
        for (int j = 0; j < L; ++j) w[u][j] = 0;
      }
      const long long row = r0 + i + u;
#pragma unroll
      for (int j = 0; j < L; ++j) {
        const float scale = e4m3_value(uint8_t(__shfl_sync(~0u, sv[u], (32 / L) * j + lane / L)));
        Dequant<T>::put(ckv_out + row * CKV + (512 / L) * j + (512 / L / 32) * lane, w[u][j], scale, ckv_scale);
      }
      Dequant<T>::put2(kpe_out + row * KPE + 2 * lane, __fmul_rn(e4m3_value(two[u] & 255), kpe_scale),
                       __fmul_rn(e4m3_value(two[u] >> 8), kpe_scale));
    }
  }
}

}  // namespace mla
