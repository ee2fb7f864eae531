// The paged KV cache in four bits (gfx950): format and addresses.
//
// Elements are E2M1 (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives), 32 dims
// share one E8M0 scale byte (2^(byte - 127); 255: the 32 dims stand for NaN).  The
// cache is [num_blocks][n_kv_heads][K, V][block_size * 68] bytes: a page holds
// block_size rows of 64 bytes (dim 2 i in the low nibble of byte i), then
// block_size rows of 4 scale bytes.  Head-major, unlike the 16-bit cache: a row of
// one token and head is only 64 bytes, half a cache line, so with the heads side by
// side every line would be fetched for two heads, each on another XCD's L2.  With
// block_size a multiple of 16 every page starts on a 64-byte boundary, a tile of 16
// tokens lies in one block, and its codes are 1 KiB and its scales 64 bytes in one
// piece.
#pragma once

#include "aac_common.h"

namespace aac {
namespace kv4 {

constexpr int kDim = 128;
constexpr int kRowBytes = 64;    // codes of a token and head
constexpr int kScaleBytes = 4;
constexpr int kTile = 16;        // tokens of a tile; block sizes are multiples of it
constexpr int kMaxBlock = 1 << 23;  // tokens of a block: offsets in its K and V pages are 32 bits

struct Cache {
  unsigned char* base;
  int64_t num_blocks;
  int32_t block_size;
  int32_t hkv;

  __host__ __device__ int64_t page_bytes() const { return (int64_t)block_size * (kRowBytes + kScaleBytes); }
  // K page of (block, head); the V page follows it
  __host__ __device__ unsigned char* page(int64_t block, int head) const {
    return base + (block * hkv + head) * 2 * page_bytes();
  }
};

// Host-side checks that every entry point shares.
inline int check_cache(const void* cache, int64_t num_blocks, int32_t block_size, int32_t hkv,
                       int32_t head_dim) {
  if (num_blocks <= 0 || block_size <= 0 || hkv <= 0) return AAC_ERR_INVALID_ARGUMENT;
  if (head_dim != kDim || block_size > kMaxBlock) return AAC_ERR_UNSUPPORTED;
  if (block_size % kTile) return AAC_ERR_SHAPE;
  if (!cache) return AAC_ERR_INVALID_ARGUMENT;
  if ((uintptr_t)cache % 64) return AAC_ERR_MISALIGNED;
  return AAC_OK;
}

}  // namespace kv4
}  // namespace aac
