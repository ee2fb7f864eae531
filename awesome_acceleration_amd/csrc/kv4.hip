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
// Sixteen lanes take a row, eight dims each, so the maximum takes two or three DPP steps.
// A group of 256 threads takes 16 consecutive tokens of two heads, so that where they
// fall into one tile of the cache (the usual case) the codes go out as 1 KiB in one
// piece.  Bound by memory: 512 bytes in (16-bit types) and 136 out a token and head.
// Measured: 32,768 tokens of 8 heads in bf16 26 us each way, 6.4 TB/s (rows that a
// prefill has just made are in the last-level cache); 262,144 tokens, stored and then loaded,
// 250 us, 5.4 TB/s, and 246, 5.5; 131,072 of fp32 6.2 and 7.1 TB/s.  The load's results go out
// with non-temporal stores (10% slower without).
#include "kv4_quant.h"

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

// How a store reads its rows: one element at a time (any alignment), 16 bytes, or 16 bytes
// past the caches.
enum class Read { Elements, Wide, Stream };

// A lane's piece of a row.
template <typename V, Read R> __device__ __forceinline__ V get(const V* p) {
  if constexpr (R == Read::Stream) return __builtin_nontemporal_load(p);
  else return *p;
}
template <Dt DT, Read R> __device__ __forceinline__ Piece<DT> load_piece(const char* row, int l) {
  Piece<DT> x;
  if constexpr (DT == Dt::FP32) {
    const float* p = reinterpret_cast<const float*>(row) + 4 * l;
    if constexpr (R != Read::Elements) {
      x.a = get<f32x4, R>(reinterpret_cast<const f32x4*>(p));
      x.b = get<f32x4, R>(reinterpret_cast<const f32x4*>(p + 64));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x.a[i] = p[i];
        x.b[i] = p[64 + i];
      }
    }
  } else if constexpr (R != Read::Elements) {
    x.w = get<u32x4, R>(reinterpret_cast<const u32x4*>(row) + l);
  } else {
    const u16* p = reinterpret_cast<const u16*>(row) + 8 * l;
#pragma unroll
    for (int i = 0; i < 4; ++i) x.w[i] = p[2 * i] | (u32)p[2 * i + 1] << 16;
  }
  return x;
}

// Heads of a workgroup, whose rows are asked for together (262,144 tokens of 8 heads, bf16, the
// store through the caches, store and load in us, each alone: one head 277 and 273, two 271
// and 238, four and eight as two).
constexpr int kHeads = 2;
constexpr int64_t kMaxGroups = 1 << 24;  // a launch's threads are numbered in 32 bits

template <Dt DT, Read R, bool PAGED>
__global__ __launch_bounds__(256) void kv4_store_kernel(StoreArgs a) {
  const int groups = (a.c.hkv + kHeads - 1) / kHeads;
  const int h0 = (int)(blockIdx.x % groups) * kHeads;
  const int64_t t = (int64_t)(blockIdx.x / groups) * 16 + (threadIdx.x >> 4);
  const int l = threadIdx.x & 15;
  if (t >= a.n_tokens) return;  // whole groups of 16 lanes
  constexpr int es = DT == Dt::FP32 ? 4 : 2;
  Piece<DT> x[kHeads][2];
#pragma unroll
  for (int h = 0; h < kHeads; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i)  // (a head past the last: the last once more, not written)
      x[h][i] = load_piece<DT, R>(a.src[i] + t * a.stride[i] + (int64_t)min(h0 + h, a.c.hkv - 1) * kDim * es, l);
  int64_t blk;
  int r;
  if constexpr (PAGED) {
    const int p = a.seqlens[t];
    if (p < 0 || p / a.c.block_size >= a.max_blocks) return;
    blk = a.block_tables[t * a.max_blocks + p / a.c.block_size];
    r = p % a.c.block_size;
    if (blk < 0 || blk >= a.c.num_blocks) return;
  } else {
    const int64_t row = a.slots[t];
    if (row < 0 || row >= a.c.num_blocks * a.c.block_size) return;
    split_row(a.c, row, &blk, &r);
  }
  unsigned char* page = a.c.page(blk, h0);
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (h0 + h >= a.c.hkv) break;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      write_row<DT>(x[h][i], l, page + r * kRowBytes,
                    reinterpret_cast<u32*>(page + a.c.block_size * kRowBytes + r * kScaleBytes));
      page += a.c.page_bytes();
    }
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
  const int groups = (a.c.hkv + kHeads - 1) / kHeads;
  const int h0 = (int)(blockIdx.x % groups) * kHeads;
  const int64_t t = (int64_t)(blockIdx.x / groups) * 16 + (threadIdx.x >> 4);
  const int l = threadIdx.x & 15;
  if (t >= a.n_tokens) return;
  const int64_t row = a.slots[t];
  const bool in = row >= 0 && row < a.c.num_blocks * a.c.block_size;
  int64_t blk;
  int r;
  split_row(a.c, in ? row : 0, &blk, &r);
  u32 w[kHeads][2], sb[kHeads][2];
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    const unsigned char* p = a.c.page(blk, min(h0 + h, a.c.hkv - 1));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned char* codes = p + r * kRowBytes;
      const unsigned char* scales = p + a.c.block_size * kRowBytes + r * kScaleBytes;
      if constexpr (DT == Dt::FP32) {
        w[h][i] = *reinterpret_cast<const u16*>(codes + 2 * l) | (u32)*reinterpret_cast<const u16*>(codes + 32 + 2 * l) << 16;
        sb[h][i] = scales[l >> 3] | (u32)scales[2 + (l >> 3)] << 8;
      } else {
        w[h][i] = *reinterpret_cast<const u32*>(codes + l * 4);
        sb[h][i] = scales[l >> 2] * 0x101u;
      }
      p += a.c.page_bytes();
    }
  }
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (h0 + h >= a.c.hkv) break;
    const int64_t at = (t * a.c.hkv + h0 + h) * kDim;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // (the scale of the first four values and of the last)
      const u32 b0 = sb[h][i] & 255u, b1 = sb[h][i] >> 8;
      const float s0 = __uint_as_float(b0 << 23), s1 = __uint_as_float(b1 << 23);
      typedef __attribute__((ext_vector_type(2))) float f2;
      f2 f[4];
      f[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[h][i], s0, 0);
      f[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[h][i], s0, 1);
      f[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[h][i], s1, 2);
      f[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[h][i], s1, 3);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = !in ? 0.f : (e < 4 ? b0 : b1) == 255u ? __uint_as_float(0x7fc00000u) : f[e >> 1][e & 1];
      if constexpr (DT == Dt::FP32) {
        f32x4* d = reinterpret_cast<f32x4*>(a.dst[i] + at * 4);
        __builtin_nontemporal_store((f32x4{x[0], x[1], x[2], x[3]}), d + l);
        __builtin_nontemporal_store((f32x4{x[4], x[5], x[6], x[7]}), d + 16 + l);
      } else {
        u32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = Elem<DT>::pack2_hw(x[2 * e], x[2 * e + 1]);
        __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(a.dst[i] + at * 2) + l);
      }
    }
  }
}

static int elem_bytes(int32_t dtype) {
  return dtype == AAC_DTYPE_FP32 ? 4 : dtype == AAC_DTYPE_BF16 || dtype == AAC_DTYPE_FP16 ? 2 : 0;
}

// Bytes of rows from which a store reads past the caches: rows that a prefill has just made
// are partly in the 256 MiB last-level cache (bf16, 8 heads, us: 32,768 tokens 26.9 and
// 31.5 past it, 262,144 273 and 258; 131,072 of fp32 234 and 207).
constexpr int64_t kStreamBytes = int64_t(512) << 20;

template <Dt DT, bool PAGED> static void launch_store_t(const StoreArgs& a, bool aligned, hipStream_t s) {
  const dim3 grid((unsigned)(cdiv(a.n_tokens, 16) * cdiv(a.c.hkv, kHeads)));
  if (!aligned) {
    hipLaunchKernelGGL((kv4_store_kernel<DT, Read::Elements, PAGED>), grid, dim3(256), 0, s, a);
    return;
  }
  if constexpr (!PAGED) {  // (an append is of one token a sequence)
    if (a.n_tokens * a.c.hkv * kDim * 2 * (DT == Dt::FP32 ? 4 : 2) >= kStreamBytes) {
      hipLaunchKernelGGL((kv4_store_kernel<DT, Read::Stream, PAGED>), grid, dim3(256), 0, s, a);
      return;
    }
  }
  hipLaunchKernelGGL((kv4_store_kernel<DT, Read::Wide, PAGED>), grid, dim3(256), 0, s, a);
}

template <bool PAGED>
static int store_common(const void* k, const void* v, int64_t k_stride, int64_t v_stride, StoreArgs a,
                        int32_t dtype, hipStream_t stream) {
  const int es = elem_bytes(dtype);
  const int64_t width = (int64_t)a.c.hkv * kDim;
  if (!k || !v) return AAC_ERR_INVALID_ARGUMENT;
  if (k_stride < width || v_stride < width) return AAC_ERR_SHAPE;
  if (((uintptr_t)k | (uintptr_t)v) % es) return AAC_ERR_MISALIGNED;
  if (cdiv(a.n_tokens, 16) * cdiv(a.c.hkv, kHeads) >= kMaxGroups) return AAC_ERR_UNSUPPORTED;
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
  if (cdiv(n_tokens, 16) * cdiv(n_kv_heads, kv4::kHeads) >= kv4::kMaxGroups) return AAC_ERR_UNSUPPORTED;
  kv4::LoadArgs a = {};
  a.c = {(unsigned char*)const_cast<void*>(cache), num_blocks, block_size, n_kv_heads};
  a.n_tokens = n_tokens;
  a.slots = slot_mapping;
  a.dst[0] = (char*)k_out;
  a.dst[1] = (char*)v_out;
  const dim3 grid((unsigned)(cdiv(n_tokens, 16) * cdiv(n_kv_heads, kv4::kHeads)));
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case AAC_DTYPE_BF16: hipLaunchKernelGGL((kv4::kv4_load_kernel<Dt::BF16>), grid, dim3(256), 0, s, a); break;
    case AAC_DTYPE_FP16: hipLaunchKernelGGL((kv4::kv4_load_kernel<Dt::FP16>), grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((kv4::kv4_load_kernel<Dt::FP32>), grid, dim3(256), 0, s, a); break;
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? AAC_OK : (int)e;
}
