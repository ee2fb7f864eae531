// Block tables and slot maps of a step from its request lengths (gfx950).
//
// Sequence b holds cached[b] tokens and gets new[b] more.  With held = ceil(cached / bs)
// and want = ceil((cached + new) / bs) - held (both within the table's width),
//   cu[b]      = sum of new over the sequences before b,
//   first[b]   = sum of want over the sequences before b,
//   table[b][held + i] = free[first[b] + i]   for i < want (-1 past the free list),
//   token i of b: position cached + i, slot table[b][position / bs] * bs + position % bs,
//                 -1 without a block.
// These are the values of paged.build_prefill_metadata (llm.py:127-140), with the
// block allocation of the host's BlockAllocator, without a byte of the maps crossing
// from the host.
//
// One launch, no workgroup waits for another: every workgroup forms both prefix sums
// for itself (8 bytes a sequence, from L2) and then takes its share of the tokens and
// of the table rows.  A new block's number is taken from the free list, not from the
// table that another workgroup may be writing.  Bound by the launch below some 100k
// tokens, then by the 16 bytes written a token.  Measured: 24 sequences of one new token
// each 3.7 us, 256 prompts 6.3.
// Lengths whose sums pass 31 bits give wrong maps, and still read and write only the
// arrays given (the comparisons with n_free below are for negative numbers too).
#include <algorithm>

#include "aac_common.h"

namespace aac {
namespace maps {

constexpr int kMaxSeqs = 8192;  // two prefix sums of ints in LDS: 64 KiB

struct Args {
  const int32_t* fresh;   // new tokens
  const int32_t* cached;  // or null: none
  int32_t* tables;
  int32_t n_seqs, width, block_size;
  const int32_t* free_blocks;  // or null: the tables are complete
  int32_t n_free;
  int64_t n_tokens;
  int32_t* cu;
  int64_t* positions;
  int64_t* slots;
  int32_t* context;
  int32_t* taken;
};

__device__ __forceinline__ int blocks_of(const Args& a, int64_t tokens) {
  return (int)min((tokens + a.block_size - 1) / a.block_size, (int64_t)a.width);
}

__global__ __launch_bounds__(256) void step_maps_kernel(Args a) {
  extern __shared__ int lds[];
  int* cu = lds;                   // [n_seqs + 1]
  int* first = lds + a.n_seqs + 1;  // [n_seqs + 1]
  __shared__ int tot[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // exclusive prefix sums, a run of consecutive sequences a thread
  const int per = (a.n_seqs + 255) / 256;
  const int b0 = min(tid * per, a.n_seqs), b1 = min(b0 + per, a.n_seqs);
  int sum[2] = {0, 0};
  for (int b = b0; b < b1; ++b) {
    const int f = max(a.fresh[b], 0), c = a.cached ? max(a.cached[b], 0) : 0;
    cu[b] = sum[0];
    first[b] = sum[1];
    sum[0] += f;
    if (a.free_blocks) sum[1] += blocks_of(a, (int64_t)c + f) - blocks_of(a, c);
  }
  int incl[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    incl[k] = sum[k];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int t = __shfl_up(incl[k], o);
      if (lane >= o) incl[k] += t;
    }
    if (lane == 63) tot[k][wave] = incl[k];
  }
  __syncthreads();
  int before[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    before[k] = incl[k] - sum[k];
    for (int w = 0; w < wave; ++w) before[k] += tot[k][w];
  }
  for (int b = b0; b < b1; ++b) {
    cu[b] += before[0];
    first[b] += before[1];
  }
  if (tid == 255) {
    cu[a.n_seqs] = before[0] + sum[0];
    first[a.n_seqs] = before[1] + sum[1];
  }
  __syncthreads();

  const int gtid = blockIdx.x * 256 + tid, gsize = gridDim.x * 256;
  for (int b = gtid; b <= a.n_seqs; b += gsize) {
    a.cu[b] = cu[b];
    if (b < a.n_seqs) a.context[b] = max(a.fresh[b], 0) + (a.cached ? max(a.cached[b], 0) : 0);
    else a.taken[0] = first[b];
  }
  if (a.free_blocks) {  // a wave a table row
    for (int b = gtid >> 6; b < a.n_seqs; b += gsize >> 6) {
      const int n = first[b + 1] - first[b];
      const int held = blocks_of(a, a.cached ? max(a.cached[b], 0) : 0);
      for (int i = lane; i < n; i += 64)
        a.tables[(int64_t)b * a.width + held + i] =
            (u32)(first[b] + i) < (u32)a.n_free ? a.free_blocks[first[b] + i] : -1;
    }
  }
  const int total = cu[a.n_seqs];
  for (int64_t i = gtid; i < a.n_tokens; i += gsize) {
    int64_t pos = 0, slot = -1;
    if (i < total) {
      int lo = 0, hi = a.n_seqs;  // cu[lo] <= i < cu[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= i) lo = mid;
        else hi = mid;
      }
      const int c = a.cached ? max(a.cached[lo], 0) : 0;
      pos = (int64_t)c + (i - cu[lo]);
      const int64_t k = pos / a.block_size;
      if (k < a.width) {
        const int held = blocks_of(a, c);
        int blk;
        if (a.free_blocks && k >= held) {
          const int64_t f = first[lo] + (k - held);
          blk = f >= 0 && f < a.n_free ? a.free_blocks[f] : -1;
        } else {
          blk = a.tables[(int64_t)lo * a.width + k];
        }
        if (blk >= 0) slot = (int64_t)blk * a.block_size + (pos - k * a.block_size);
      }
    }
    a.positions[i] = pos;
    a.slots[i] = slot;
  }
}

}  // namespace maps
}  // namespace aac

using namespace aac;

extern "C" int aac_step_maps(const int32_t* new_lens, const int32_t* cached_lens, int32_t* block_tables,
                             int32_t n_seqs, int32_t max_blocks_per_seq, int32_t block_size,
                             const int32_t* free_blocks, int32_t n_free, int64_t n_tokens,
                             int32_t* cu_seqlens, int64_t* positions, int64_t* slot_mapping,
                             int32_t* context_lens, int32_t* blocks_taken, void* stream) {
  if (n_seqs < 0 || max_blocks_per_seq <= 0 || block_size <= 0 || n_free < 0 || n_tokens < 0)
    return AAC_ERR_INVALID_ARGUMENT;
  if (n_seqs > maps::kMaxSeqs || n_tokens > 0x7fffffff) return AAC_ERR_UNSUPPORTED;
  if (!cu_seqlens || !blocks_taken || (n_tokens && (!positions || !slot_mapping)))
    return AAC_ERR_INVALID_ARGUMENT;
  if (n_seqs && (!new_lens || !block_tables || !context_lens)) return AAC_ERR_INVALID_ARGUMENT;
  if (n_free && !free_blocks) return AAC_ERR_INVALID_ARGUMENT;
  maps::Args a = {};
  a.fresh = new_lens;
  a.cached = cached_lens;
  a.tables = block_tables;
  a.n_seqs = n_seqs;
  a.width = max_blocks_per_seq;
  a.block_size = block_size;
  a.free_blocks = free_blocks;
  a.n_free = n_free;
  a.n_tokens = n_tokens;
  a.cu = cu_seqlens;
  a.positions = positions;
  a.slots = slot_mapping;
  a.context = context_lens;
  a.taken = blocks_taken;
  const int64_t most = std::max<int64_t>(n_tokens, (int64_t)n_seqs * 64);
  const unsigned grid = (unsigned)std::min<int64_t>(std::max<int64_t>(cdiv(most, 256), 1), 1024);
  hipLaunchKernelGGL(maps::step_maps_kernel, dim3(grid), dim3(256), (size_t)(n_seqs + 1) * 8,
                     (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? AAC_OK : (int)e;
}
