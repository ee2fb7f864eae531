// 4-bit KV cache: store, append and load (gfx950).  Format: kv4.h.
//
// Store.  For each token, KV head and 32 dims x[0..31] of a K or V row, with
// a = max |x|:
//   e    = exponent of a rounded to two significant bits, minus 2 (the exponent of
//          the largest code, 6), within [-125, 125];
//   code = x / 2^e rounded to the E2M1 grid, halves to the even code, at most 6;
//   byte = e + 127, or 255 with codes 0 where a is infinite or NaN.
// Rounding a up from 1.75 x 2^n on keeps the largest value within half a step: it
// becomes 4 x 2^(n - 1), not 6 x 2^(n - 2) a quarter below it.  The division by a
// power of two is exact, and v_cvt_scalef32_pk_fp4_f32 does it with the rounding.
// The bounds of e keep every value a normal number of bfloat16.
//
// Sixteen lanes take a row, eight dims each; four of them share a scale, so the
// maximum takes two DPP steps.  A group of 256 threads takes 16 consecutive tokens of
// one head, so that where they fall into one tile of the cache (the usual case) the
// codes go out as 1 KiB in one piece.  Bound by memory: 512 bytes in (16-bit types)
// and 136 out a token and head.
#include "kv4.h"

namespace aac {
namespace kv4 {

struct StoreArgs {
  const char* src[2];   // k, v
  int64_t stride[2];    // bytes between tokens
  Cache c;
  int64_t n_tokens;
  const int64_t* slots;         // store
  const int32_t* block_tables;  // append
  const int32_t* seqlens;
  int32_t max_blocks;
};

template <Dt DT> __device__ __forceinline__ float elem_f32(const char* p);
template <> __device__ __forceinline__ float elem_f32<Dt::BF16>(const char* p) {
  return bf16lo(*reinterpret_cast<const u16*>(p));
}
template <> __device__ __forceinline__ float elem_f32<Dt::FP16>(const char* p) {
  return (float)*reinterpret_cast<const _Float16*>(p);
}
template <> __device__ __forceinline__ float elem_f32<Dt::FP32>(const char* p) {
  return *reinterpret_cast<const float*>(p);
}

// eight elements of a row as float
template <Dt DT, bool ALIGNED> __device__ __forceinline__ void load8(const char* p, float* x) {
  constexpr int es = DT == Dt::FP32 ? 4 : 2;
  if constexpr (!ALIGNED) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = elem_f32<DT>(p + i * es);
  } else if constexpr (DT == Dt::FP32) {
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else {
    Elem<DT>::unpack8(*reinterpret_cast<const u32x4*>(p), x);
  }
}

// codes of eight elements; the four lanes of a quad hold the 32 of a scale
__device__ __forceinline__ u32 quantise8(const float* x, u32* scale_byte) {
  u32 a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(x[i]) & 0x7fffffffu);
  a = max(a, (u32)__builtin_amdgcn_update_dpp(0, (int)a, kDppQuadXor1, 0xF, 0xF, false));
  a = max(a, (u32)__builtin_amdgcn_update_dpp(0, (int)a, kDppQuadXor2, 0xF, 0xF, false));
  const bool bad = a >= 0x7f800000u;
  const int e = min(max((int)((a + 0x200000u) >> 23) - 2, 2), 252);
  const float s = __uint_as_float((u32)e << 23);
  u32 w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  *scale_byte = bad ? 255u : (u32)e;
  return bad ? 0u : w;
}

template <Dt DT, bool ALIGNED, bool PAGED>
__global__ __launch_bounds__(256) void kv4_store_kernel(StoreArgs a) {
  const int h = blockIdx.x % a.c.hkv;
  const int64_t t = (int64_t)(blockIdx.x / a.c.hkv) * 16 + (threadIdx.x >> 4);
  const int l = threadIdx.x & 15;
  if (t >= a.n_tokens) return;  // whole groups of 16 lanes
  int64_t row;
  if constexpr (PAGED) {
    const int p = a.seqlens[t];
    if (p < 0 || p / a.c.block_size >= a.max_blocks) return;
    const int blk = a.block_tables[t * a.max_blocks + p / a.c.block_size];
    if (blk < 0 || blk >= a.c.num_blocks) return;
    row = (int64_t)blk * a.c.block_size + p % a.c.block_size;
  } else {
    row = a.slots[t];
    if (row < 0 || row >= a.c.num_blocks * a.c.block_size) return;
  }
  const int64_t blk = row / a.c.block_size;
  const int r = (int)(row - blk * a.c.block_size);
  constexpr int es = DT == Dt::FP32 ? 4 : 2;
  float x[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    load8<DT, ALIGNED>(a.src[i] + t * a.stride[i] + (h * kDim + l * 8) * es, x[i]);
  unsigned char* page = a.c.page(blk, h);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    u32 sb;
    const u32 w = quantise8(x[i], &sb);
    *reinterpret_cast<u32*>(page + r * kRowBytes + l * 4) = w;
    if ((l & 3) == 0) page[a.c.block_size * kRowBytes + r * kScaleBytes + (l >> 2)] = (unsigned char)sb;
    page += a.c.page_bytes();
  }
}

struct LoadArgs {
  Cache c;
  int64_t n_tokens;
  const int64_t* slots;
  char* dst[2];  // [n, hkv, 128] each
};

template <Dt DT>
__global__ __launch_bounds__(256) void kv4_load_kernel(LoadArgs a) {
  const int h = blockIdx.x % a.c.hkv;
  const int64_t t = (int64_t)(blockIdx.x / a.c.hkv) * 16 + (threadIdx.x >> 4);
  const int l = threadIdx.x & 15;
  if (t >= a.n_tokens) return;
  const int64_t row = a.slots[t];
  const bool in = row >= 0 && row < a.c.num_blocks * a.c.block_size;
  const int64_t blk = in ? row / a.c.block_size : 0;
  const int r = in ? (int)(row - blk * a.c.block_size) : 0;
  const unsigned char* page = a.c.page(blk, h);
  u32 w[2], sb[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const unsigned char* p = page + i * a.c.page_bytes();
    w[i] = *reinterpret_cast<const u32*>(p + r * kRowBytes + l * 4);
    sb[i] = p[a.c.block_size * kRowBytes + r * kScaleBytes + (l >> 2)];
  }
  const int64_t at = (t * a.c.hkv + h) * kDim + l * 8;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float s = __uint_as_float(sb[i] << 23);
    typedef __attribute__((ext_vector_type(2))) float f2;
    f2 f[4];
    f[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 0);
    f[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 1);
    f[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 2);
    f[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], s, 3);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = !in ? 0.f : sb[i] == 255u ? __uint_as_float(0x7fc00000u) : f[e >> 1][e & 1];
    if constexpr (DT == Dt::FP32) {
      f32x4* d = reinterpret_cast<f32x4*>(a.dst[i] + at * 4);
      d[0] = f32x4{x[0], x[1], x[2], x[3]};
      d[1] = f32x4{x[4], x[5], x[6], x[7]};
    } else {
      u32x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = Elem<DT>::pack2_hw(x[2 * e], x[2 * e + 1]);
      *reinterpret_cast<u32x4*>(a.dst[i] + at * 2) = o;
    }
  }
}

static int elem_bytes(int32_t dtype) {
  return dtype == AAC_DTYPE_FP32 ? 4 : dtype == AAC_DTYPE_BF16 || dtype == AAC_DTYPE_FP16 ? 2 : 0;
}

template <Dt DT, bool PAGED> static void launch_store_t(const StoreArgs& a, bool aligned, hipStream_t s) {
  const dim3 grid((unsigned)(cdiv(a.n_tokens, 16) * a.c.hkv));
  if (aligned)
    hipLaunchKernelGGL((kv4_store_kernel<DT, true, PAGED>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((kv4_store_kernel<DT, false, PAGED>), grid, dim3(256), 0, s, a);
}

template <bool PAGED>
static int store_common(const void* k, const void* v, int64_t k_stride, int64_t v_stride, StoreArgs a,
                        int32_t dtype, hipStream_t stream) {
  const int es = elem_bytes(dtype);
  const int64_t width = (int64_t)a.c.hkv * kDim;
  if (!k || !v) return AAC_ERR_INVALID_ARGUMENT;
  if (k_stride < width || v_stride < width) return AAC_ERR_SHAPE;
  if (((uintptr_t)k | (uintptr_t)v) % es) return AAC_ERR_MISALIGNED;
  if (cdiv(a.n_tokens, 16) * a.c.hkv > 0x7fffffff) return AAC_ERR_SHAPE;
  a.src[0] = (const char*)k;
  a.src[1] = (const char*)v;
  a.stride[0] = k_stride * es;
  a.stride[1] = v_stride * es;
  const bool aligned = (((uintptr_t)k | (uintptr_t)v) % 16) == 0 && (a.stride[0] | a.stride[1]) % 16 == 0;
  switch (dtype) {
    case AAC_DTYPE_BF16: launch_store_t<Dt::BF16, PAGED>(a, aligned, stream); break;
    case AAC_DTYPE_FP16: launch_store_t<Dt::FP16, PAGED>(a, aligned, stream); break;
    default: launch_store_t<Dt::FP32, PAGED>(a, aligned, stream); break;
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? AAC_OK : (int)e;
}

}  // namespace kv4
}  // namespace aac

using namespace aac;

extern "C" int aac_kv4_store(const void* k, const void* v, int64_t k_tok_stride, int64_t v_tok_stride,
                             void* cache, int64_t num_blocks, int32_t block_size,
                             const int64_t* slot_mapping, int64_t n_tokens, int32_t n_kv_heads,
                             int32_t head_dim, int32_t dtype, void* stream) {
  if (!kv4::elem_bytes(dtype)) return AAC_ERR_UNSUPPORTED;
  if (n_tokens < 0) return AAC_ERR_INVALID_ARGUMENT;
  if (n_tokens == 0) return AAC_OK;
  const int rc = kv4::check_cache(cache, num_blocks, block_size, n_kv_heads, head_dim);
  if (rc != AAC_OK) return rc;
  if (!slot_mapping) return AAC_ERR_INVALID_ARGUMENT;
  kv4::StoreArgs a = {};
  a.c = {(unsigned char*)cache, num_blocks, block_size, n_kv_heads};
  a.n_tokens = n_tokens;
  a.slots = slot_mapping;
  return kv4::store_common<false>(k, v, k_tok_stride, v_tok_stride, a, dtype, (hipStream_t)stream);
}

extern "C" int aac_kv4_append(const void* k, const void* v, int64_t k_seq_stride, int64_t v_seq_stride,
                              void* cache, int64_t num_blocks, int32_t block_size,
                              const int32_t* block_tables, int32_t max_blocks_per_seq,
                              const int32_t* cache_seqlens, int32_t n_seqs, int32_t n_kv_heads,
                              int32_t head_dim, int32_t dtype, void* stream) {
  if (!kv4::elem_bytes(dtype)) return AAC_ERR_UNSUPPORTED;
  if (n_seqs < 0 || max_blocks_per_seq <= 0) return AAC_ERR_INVALID_ARGUMENT;
  if (n_seqs == 0) return AAC_OK;
  const int rc = kv4::check_cache(cache, num_blocks, block_size, n_kv_heads, head_dim);
  if (rc != AAC_OK) return rc;
  if (!block_tables || !cache_seqlens) return AAC_ERR_INVALID_ARGUMENT;
  kv4::StoreArgs a = {};
  a.c = {(unsigned char*)cache, num_blocks, block_size, n_kv_heads};
  a.n_tokens = n_seqs;
  a.block_tables = block_tables;
  a.seqlens = cache_seqlens;
  a.max_blocks = max_blocks_per_seq;
  return kv4::store_common<true>(k, v, k_seq_stride, v_seq_stride, a, dtype, (hipStream_t)stream);
}

extern "C" int aac_kv4_load(const void* cache, int64_t num_blocks, int32_t block_size,
                            const int64_t* slot_mapping, int64_t n_tokens, int32_t n_kv_heads,
                            int32_t head_dim, void* k_out, void* v_out, int32_t dtype, void* stream) {
  if (!kv4::elem_bytes(dtype)) return AAC_ERR_UNSUPPORTED;
  if (n_tokens < 0) return AAC_ERR_INVALID_ARGUMENT;
  if (n_tokens == 0) return AAC_OK;
  const int rc = kv4::check_cache(cache, num_blocks, block_size, n_kv_heads, head_dim);
  if (rc != AAC_OK) return rc;
  if (!slot_mapping || !k_out || !v_out) return AAC_ERR_INVALID_ARGUMENT;
  if (((uintptr_t)k_out | (uintptr_t)v_out) % 16) return AAC_ERR_MISALIGNED;
  if (cdiv(n_tokens, 16) * n_kv_heads > 0x7fffffff) return AAC_ERR_SHAPE;
  kv4::LoadArgs a = {};
  a.c = {(unsigned char*)const_cast<void*>(cache), num_blocks, block_size, n_kv_heads};
  a.n_tokens = n_tokens;
  a.slots = slot_mapping;
  a.dst[0] = (char*)k_out;
  a.dst[1] = (char*)v_out;
  const dim3 grid((unsigned)(cdiv(n_tokens, 16) * n_kv_heads));
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case AAC_DTYPE_BF16: hipLaunchKernelGGL((kv4::kv4_load_kernel<Dt::BF16>), grid, dim3(256), 0, s, a); break;
    case AAC_DTYPE_FP16: hipLaunchKernelGGL((kv4::kv4_load_kernel<Dt::FP16>), grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((kv4::kv4_load_kernel<Dt::FP32>), grid, dim3(256), 0, s, a); break;
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? AAC_OK : (int)e;
}
