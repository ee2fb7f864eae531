// Combining the partial results of a context that was split over workgroups
// (gfx950); shared by the paged decode kernels.
#pragma once

#include "aac_common.h"

namespace aac {

template <Dt DT>
__device__ __forceinline__ void store_out2(void* out, int64_t idx, float x0, float x1) {
  if constexpr (DT == Dt::FP32) {
    *reinterpret_cast<float2*>(reinterpret_cast<float*>(out) + idx) = make_float2(x0, x1);
  } else {
    *reinterpret_cast<u32*>(reinterpret_cast<u16*>(out) + idx) = Elem<DT>::pack2(x0, x1);
  }
}

// The partitions of one (sequence, query head), rows slot0 .. slot0 + np - 1 of 128
// dims each: out = sum_p 2^(lse_p - LSE) o_p with LSE = log2 sum_p 2^lse_p.
// Four wavefronts per (sequence, query head): each finds the largest lse (one
// load per 64 partitions), then wave w sums partitions w, w + 4, ... with four
// in flight, and the four sums meet in LDS.  The chain of loads is what it
// costs: one wave walking the partitions one by one took 5.2 us at 11 partitions
// of 24 sequences.
template <Dt DT>
__device__ __forceinline__ void combine_partitions(const float* ws_o, const float* ws_lse, int64_t slot0,
                                                   int np, void* out, int64_t out_at) {
  constexpr int kDims = 128;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float mx = -INFINITY;
  for (int p = lane; p < np; p += 64) mx = fmaxf(mx, ws_lse[slot0 + p]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
  float W = 0.f, o0 = 0.f, o1 = 0.f;
  for (int p = wave; p < np; p += 16) {
    float lse[4];
    float2 o[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t slot = slot0 + min(p + 4 * u, np - 1);
      lse[u] = ws_lse[slot];
      o[u] = *reinterpret_cast<const float2*>(ws_o + slot * kDims + 2 * lane);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      // past the end: nothing, not 0 x the last partition's (infinite?) result
      const bool in = p + 4 * u < np;
      const float w = fast_exp2(lse[u] - mx);
      W += in ? w : 0.f;
      o0 = in ? fmaf(w, o[u].x, o0) : o0;
      o1 = in ? fmaf(w, o[u].y, o1) : o1;
    }
  }
  __shared__ float sw[4];
  __shared__ float2 so[4][64];
  so[wave][lane] = make_float2(o0, o1);
  if (lane == 0) sw[wave] = W;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    W += sw[w];
    o0 += so[w][lane].x;
    o1 += so[w][lane].y;
  }
  const float inv = 1.f / W;
  store_out2<DT>(out, out_at + 2 * lane, o0 * inv, o1 * inv);
}

}  // namespace aac
