// Decode attention over the 4-bit paged KV cache (gfx950).  Format: kv4.h.
//
//   out[b, hq] = sum_t softmax_t(scale q[b, hq] . k_t) v_t,   t < context of b
//
// A workgroup takes one KV head's group of G <= 16 query heads over one partition of
// a sequence's tokens; its four waves take steps of 64 tokens in turn and keep an
// online softmax each (log2 domain), merged at the end; partitions are combined by
// a second launch.  Steps in turn, not a quarter of the partition each: the workgroup
// then reads pages in order, and the waves end together.
//
// Both products run on v_mfma_f32_16x16x32_bf16.  A cached value is a 2-bit significand
// times a power of two, so its bfloat16 is exact (v_cvt_scalef32_pk_bf16_fp4: two
// values an instruction, the scale included).  What is rounded is the other operand:
//   queries are split in 1, 2 or 3 bfloat16 terms (bf16, fp16, fp32), probabilities in 2,
//   2 or 3, one product for each: queries are exact, and what is cut off a probability is
//   below 2^-14 of it, in fp32 2^-21.  (A bf16 call's probabilities rounded to one term take 1 to 3%
//   less time - the first case below 73 us against 75, the second 281 against 285 -
//   and leave an output 0.0020 off where its own rounding alone is 0.0017.)
// Sums, the running maximum and the partial results are float.
//
// Scores are computed transposed, S^T = K Q^T: lane (t = lane % 16, j = lane / 16)
// reads 16 bytes of token t's codes, dims 32 j .. 32 j + 31, which is one scale and
// (in four instructions of 8 dims) the K operand.  The result has query lane % 16
// and tokens 4 j .. 4 j + 3 in each lane, which is, for two tiles of 16 tokens, the P
// operand of O^T += V^T P^T with tokens in the order (tile, 4 j + i).  V^T needs four
// tokens of one dim a lane: V is converted in token order like K, written to the
// wave's own 8 KiB of LDS as bf16 and read back with the transposing load
// ds_read_b64_tr_b16.  Slots of 16 bytes sit at slot ^ (2 (row & 7) | row >> 3), with
// which neither the b128 writes nor the transposing reads meet a bank twice.  Scales
// (256 bytes of K and of V a step) go through LDS too: one dword a lane and page
// instead of a byte a lane for each tile.
//
// Bound by the way the rows arrive: with the arithmetic left out, the loads alone take
// 69.7, 276 and 28 us of the cases below, and the arithmetic alone (rows held, one term of the
// probabilities) 50, 198.
// So rows are asked for where the last ones have been taken, a step ahead of their use
// (deeper rings spill or lose a workgroup a CU, and gained nothing), as non-temporal buffer loads, whose
// bounds stand for the branch at a partition's end, 1 KiB of codes in one piece each.
// Measured on MI355X (GPU time): bf16, 256 sequences of 1,024 to 2,048 tokens, 16/8 heads
// 75 us (the bytes alone, at the 7.0 TB/s of a large copy: 61); 64 of 16,384 to 32,768
// 285 (244); fp16, one of 115,000 32 (19), of which the second launch is 4; fp32, 4 of up
// to 400 tokens 7.7, where latency alone counts.
#include <algorithm>
#include <climits>

#include "decode_reduce.h"
#include "kv4.h"

namespace aac {
namespace kv4 {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;
typedef __attribute__((address_space(3))) unsigned char lds_u8;
typedef unsigned long long u64;

constexpr int64_t kMaxContext = (int64_t(1) << 31) - 1024;  // tokens: the steps' numbers stay within 31 bits
constexpr float kRescale = 8.f;  // probabilities up to 2^8 before the reference moves

struct DecArgs {
  const void* q;
  int64_t q_stride;  // elements
  Cache c;
  const int32_t* block_tables;
  int32_t max_blocks;
  const int32_t* lens;
  int32_t lens_add;
  int32_t n_seqs, hq, g;
  float scale_log2;
  void* out;
  int64_t out_stride;
  int32_t n_parts, part_tokens;
  // The plan's rule by a context's own length, for those far below the capacity (part_of):
  int32_t tight;       // from here on partitions of part_tokens
  int32_t whole;       // up to here no split
  uint64_t per_round;  // items / those of a round of workgroups, 16 bits of fraction
  u32 inv_parts;       // 2^32 / n_parts, rounded up
  float* ws_o;    // [n_seqs, hq, n_parts, 128]
  float* ws_lse;  // [n_seqs, hq, n_parts]
  // tile number -> block: (tile * magic) >> shift
  uint64_t magic;
  int32_t shift;
  int32_t alone;      // the longest context that one wave takes
};

constexpr int kStep = 64;         // tokens of a step
constexpr int kTurn = 4 * kStep;  // of one turn of the workgroup's waves

__host__ __device__ __forceinline__ int cdiv_turn(int tokens) { return (tokens + kTurn - 1) / kTurn * kTurn; }
// A partition, from what one round of workgroups makes of all tokens (plan)
__host__ __device__ __forceinline__ u32 rounds_part(u32 round) {
  return round <= 1024 ? round : round <= 4096 ? 1024 : round <= 8192 ? 2048 : 4096;
}

__device__ __forceinline__ int context_len(const DecArgs& a, int len) {
  const int64_t ctx = (int64_t)len + a.lens_add;
  const int64_t cap = min((int64_t)a.max_blocks * a.c.block_size, kMaxContext);
  return (int)(ctx < 0 ? 0 : ctx > cap ? cap : ctx);
}
// Tokens of a partition of a context.  The plan sizes them for the largest context that
// there may be; one that would fill less than a quarter of its partitions (of a captured
// step, mostly) is split by the same rule for its own length, never coarser and into
// no more than n_parts (us, with its own length and with the plan's partitions, at 8
// heads: 16 x 500-2,000 in tables of 32,768 16.0 and 20.9, 32 of them 18.4 and 25.3, 8 x 3-30k
// in 131,072 29.6 and 53.6; without the quarter 100 x 2-6k in 6,000 took 93, not 83).
__device__ __forceinline__ int part_of(const DecArgs& a, int ctx) {
  if (ctx >= a.tight) return a.part_tokens;
  int part = ctx;
  if (ctx > a.whole) {
    const u32 round = (u32)min((u64)(u32)ctx * a.per_round >> 16, (u64)(1u << 30));
    const u32 least = (u32)(((u64)(u32)(ctx - 1) * a.inv_parts) >> 32) + 1;
    part = (int)max(max(rounds_part(round), (u32)ctx >> 6), least);
  }
  return min(cdiv_turn(max(part, 1)), a.part_tokens);
}
__device__ __forceinline__ int parts_of(const DecArgs& a, int ctx, int part_tokens) {
  return min(a.n_parts, (int)(((u32)ctx + (u32)part_tokens - 1) / (u32)part_tokens));
}

// The high halves of two floats as a bf16 pair, and what is left of each
__device__ __forceinline__ u32 take_bf16(float& x, float& y) {
  const u32 w = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), kSelHi);
  x -= __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  y -= __uint_as_float(__float_as_uint(y) & 0xffff0000u);
  return w;
}

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                 c, 0, 0, 0);
}

// eight codes (a dword) times 2^(byte - 127), as bf16
__device__ __forceinline__ u32x4 values8(u32 w, float scale) {
  return u32x4{__builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
               __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
               __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
               __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
}

// One step's codes of a lane, K and V of four tiles, and the scales of one token each.
struct Raw {
  u32x4 k[4], v[4];
  u32 ks, vs;
};

constexpr int kLoadAux = 2;  // non-temporal: nothing reads the rows again

// WIDE: block sizes are a multiple of a step, so that a step lies in one block.
template <Dt DT, bool WIDE>
__global__ __launch_bounds__(256, DT == Dt::FP32 ? 2 : 3) void kv4_decode_kernel(DecArgs a) {
  // terms of a query and of a probability
  constexpr int NT = DT == Dt::BF16 ? 1 : DT == Dt::FP16 ? 2 : 3, NP = DT == Dt::FP32 ? 3 : 2;
  constexpr int kWaveLds = 32 * 256;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4 * kWaveLds];
  __shared__ u32 s_scale[4][2][kStep];
  __shared__ float sm_m[4][16], sm_l[4][16];
  const int part = blockIdx.y, b = blockIdx.z;
  int h = blockIdx.x;
  if (part >= a.n_parts) return;  // (the one that makes their number odd)
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, j = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  typedef const int32_t __attribute__((address_space(4))) cint;  // scalar loads
  const cint* table = (const cint*)(uintptr_t)(a.block_tables + (int64_t)b * a.max_blocks);
  const int tpb = a.c.block_size / kTile;
  constexpr int kLooks = WIDE ? 1 : 4;
  struct Where {
    int block[kLooks], row[kLooks];  // of a step's tiles: table entry, first row in the block
  };
  auto look = [&](int t0, int tiles, Where& w) {
#pragma unroll
    for (int k = 0; k < kLooks; ++k) {
      // past the end: the last again (its first tile where one look serves a whole step,
      // whose rows then all lie in the block)
      const int tile = min(t0 / kTile + k, WIDE ? (tiles - 1) & ~(kStep / kTile - 1) : tiles - 1);
      const int bi = (int)(((u64)(u32)tile * a.magic) >> a.shift);
      w.block[k] = table[bi];
      w.row[k] = (tile - bi * tpb) * kTile;
    }
  };
  const int ctx = context_len(a, ((const cint*)(uintptr_t)a.lens)[b]);
  const int part_tokens = part_of(a, ctx);
  const int np = parts_of(a, ctx, part_tokens);
  if (part >= np) {  // workgroup-uniform
    if (part == 0) {  // an empty context
      for (int i = tid; i < a.g * (kDim / 2); i += 256)
        store_out2<DT>(a.out, (int64_t)b * a.out_stride + (int64_t)h * a.g * kDim + 2 * i, 0.f, 0.f);
    }
    return;
  }
  // A short context of many: each of the group's waves takes a head to itself, and three of
  // four workgroups end here.  Which one stays moves on from sequence to sequence, and
  // once more every fourth: workgroups go round the XCDs and their shader engines in turn,
  // and every fourth would meet the same engine.
  const bool alone = ctx <= a.alone;
  if (alone) {
    if ((h ^ (b + (b >> 2))) & 3) return;
    h = (h & ~3) + wave;
  }
  // The waves take steps in turn.
  const int beg = part * part_tokens, t_first = alone ? 0 : beg + kStep * wave, stride = alone ? kStep : kTurn;
  const int end = beg + min(ctx - beg, part_tokens), n_tiles = (end + kTile - 1) / kTile;

  // A buffer of each tile's pages (K, then V) from the block number, and offsets that each
  // lane keeps.  Past the end the buffer is empty: the loads are issued all the same, so
  // that the number in flight is known, and read nothing.
  const int pb = (int)a.c.page_bytes();
  const int voff = n * kRowBytes + 16 * j;
  auto page_of = [&](int block) { return a.c.page((u32)block < (u32)a.c.num_blocks ? (u32)block : 0u, h); };
  auto load_codes = [&](int t0, const Where& w, int k, bool v) {
    const __amdgpu_buffer_rsrc_t page = __builtin_amdgcn_make_buffer_rsrc(
        page_of(w.block[WIDE ? 0 : k]), 0, t0 + (WIDE ? 0 : kTile * k) < end ? 2 * pb : 0, 0x00020000);
    const int row = WIDE ? w.row[0] + kTile * k : w.row[k];
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                         page, voff, (v ? pb : 0) + row * kRowBytes, kLoadAux));
  };
  // lane l: the four scales of token l of the step (of the last tile's past the end)
  auto load_scales = [&](const Where& w, Raw& r) {
    uint64_t at = 0;
#pragma unroll
    for (int k = 0; k < kLooks; ++k) {
      const uint64_t t = (uint64_t)page_of(w.block[k]) + (u32)(a.c.block_size * kRowBytes + w.row[k] * kScaleBytes);
      at = k == 0 || j == k ? t : at;
    }
    // (a global address: a flat load would also count as an LDS access)
    typedef const __attribute__((address_space(1))) u32 gu32;
    const uint64_t p = at + (u32)((WIDE ? lane : n) * kScaleBytes);
    r.ks = __builtin_nontemporal_load((gu32*)p);
    r.vs = __builtin_nontemporal_load((gu32*)(p + (u32)pb));
  };
  // One buffer of rows: those of the next step are asked for where this step's have been
  // taken.
  Raw r;
  Where w;
  look(t_first, n_tiles, w);
  load_scales(w, r);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    r.k[k] = load_codes(t_first, w, k, false);
    r.v[k] = load_codes(t_first, w, k, true);
  }

  // Q operand: query n's dims 32 j + 8 i .. + 7 for product i, in NT terms
  // (a negative scale: -q and -scale, so that the largest product has the largest score)
  const float cs = vmax(fabsf(a.scale_log2), 1e-30f);  // (a scale of 0: equal scores; NaN stays)
  u32x4 qf[NT][4];
  {
    const bool row = n < a.g;
    const u32 flip = a.scale_log2 < 0.f ? 0x80000000u : 0u, keep = row ? 0xffffffffu : 0u;
    const int64_t at = (int64_t)b * a.q_stride + (int64_t)(h * a.g + (row ? n : 0)) * kDim + 32 * j;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == Dt::BF16) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(reinterpret_cast<const u16*>(a.q) + at + 8 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) qf[0][i][e] = (w[e] ^ (flip | flip >> 16)) & keep;
      } else {
        float x[8];
        if constexpr (DT == Dt::FP16) {
          Elem<DT>::unpack8(*reinterpret_cast<const u32x4*>(reinterpret_cast<const u16*>(a.q) + at + 8 * i), x);
        } else {
          const f32x4* p = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(a.q) + at + 8 * i);
          const f32x4 lo = p[0], hi = p[1];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e] = lo[e];
            x[4 + e] = hi[e];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __uint_as_float((__float_as_uint(x[e]) ^ flip) & keep);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) qf[t][i][e] = take_bf16(x[2 * e], x[2 * e + 1]);
      }
    }
  }

  lds_u8* vb = (lds_u8*)lds + wave * kWaveLds;
  // writes: token n's dims 32 j + 8 i, 16-byte slot 4 j + i of its row; reads: this
  // quarter's tokens 4 j + (n >> 2), dims 16 d + 4 (n & 3), slot 2 d + (n & 3) / 2
  auto swizzle = [](int row) { return ((row & 7) << 1) | (row >> 3); };
  const int wt = n * 256 + ((4 * j ^ swizzle(n)) << 4);
  const int rt = 4 * j + (n >> 2), rd = rt * 256 + ((((n & 3) >> 1) ^ swizzle(rt)) << 4) + 8 * (n & 1);
  f32x4 o[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  // running maximum of q . k, the exponents' reference (cs times it; 0 while it is -inf),
  // lane-partial sum
  float m = -INFINITY, ref = 0.f, l = 0.f;
  const float margin = kRescale / cs;

  look(t_first + stride, n_tiles, w);
  // The scales have arrived before the loop: with them among the loads under way at its
  // entry, the compiler waits for every load at its top (the counts of both ways in
  // have to agree).
  asm volatile("" : "+v"(r.ks), "+v"(r.vs));
  __attribute__((address_space(3))) u32* sc = (__attribute__((address_space(3))) u32*)&s_scale[wave][0][0];
  const __attribute__((address_space(3))) unsigned char* sc8 =
      (const __attribute__((address_space(3))) unsigned char*)&s_scale[wave][0][0] + n * kScaleBytes + j;
  for (int t0 = t_first; t0 < end; t0 += stride) {
    sc[lane] = r.ks;
    sc[kStep + lane] = r.vs;
    asm volatile("" ::: "memory");
    load_scales(w, r);
    f32x4 s[4];
    u32 vs[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      s[k] = f32x4{0.f, 0.f, 0.f, 0.f};
      const float ks = __uint_as_float((u32)sc8[k * 64] << 23);
      vs[k] = sc8[kStep * kScaleBytes + k * 64];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x4 kf = values8(r.k[k][i], ks);
#pragma unroll
        for (int x = 0; x < NT; ++x) s[k] = mfma(kf, qf[x][i], s[k]);
      }
      // (kept here: asked for earlier, the rows need registers of their own and a copy)
      __builtin_amdgcn_sched_barrier(0);
      r.k[k] = load_codes(t0 + stride, w, k, false);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (t0 + kStep > end) {  // the last rows: those past the end stand for nothing
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t0 + 16 * k + 4 * j + i >= end) s[k][i] = -INFINITY;
        if (t0 + 16 * k + n >= end) {  // (their bytes may stand for NaN)
          r.v[k] = u32x4{0, 0, 0, 0};
          vs[k] = 127;
        }
      }
    }
    float mx = vmax3(vmax3(s[0][0], s[0][1], s[0][2]), s[0][3], s[1][0]);
    mx = vmax3(vmax3(mx, s[1][1], s[1][2]), s[1][3], s[2][0]);
    mx = vmax3(vmax3(mx, s[2][1], s[2][2]), s[2][3], s[3][0]);
    mx = vmax(vmax3(mx, s[3][1], s[3][2]), s[3][3]);
    if (__ballot(mx > m + margin)) {
      mx = vmax(mx, __shfl_xor(mx, 16));
      mx = vmax(mx, __shfl_xor(mx, 32));
      const bool none = m == -INFINITY;  // nothing is summed yet
      m = vmax(m, mx);
      const float to = m == -INFINITY ? 0.f : m * cs;
      const float f = none ? 0.f : fast_exp2(ref - to);
      ref = to;
      l *= f;
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][i] *= f;
    }
    u32x4 pf[2][NP];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        u32x4* const p = pf[k >> 1];
        const int at = 2 * (k & 1) + e;
        float x = fast_exp2(fmaf(s[k][2 * e], cs, -ref)), y = fast_exp2(fmaf(s[k][2 * e + 1], cs, -ref));
        l += x + y;
#pragma unroll
        for (int c = 0; c < NP; ++c) p[c][at] = take_bf16(x, y);
      }
#pragma unroll
    for (int q = 0; q < 2; ++q) {  // 32 tokens
      // (fp16: the addresses formed anew, 16 registers for a third workgroup per CU)
      int wo = wt, ro = rd;
      if constexpr (NT == 2) asm volatile("" : "+v"(wo), "+v"(ro));
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float sv = __uint_as_float(vs[2 * q + k] << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(vb + (wo ^ i * 16) + k * 4096) =
              values8(r.v[2 * q + k][i], sv);
        __builtin_amdgcn_sched_barrier(0);
        r.v[2 * q + k] = load_codes(t0 + stride, w, 2 * q + k, true);
        __builtin_amdgcn_sched_barrier(0);
      }
      asm volatile("" ::: "memory");
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(vb + (ro ^ d * 32)));
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(vb + (ro ^ d * 32) + 16 * 256));
        const u32x2 a0 = __builtin_bit_cast(u32x2, lo), a1 = __builtin_bit_cast(u32x2, hi);
        const u32x4 vf = {a0[0], a0[1], a1[0], a1[1]};
#pragma unroll
        for (int c = 0; c < NP; ++c) o[d] = mfma(vf, pf[q][c], o[d]);
      }
      asm volatile("" ::: "memory");
    }
    look(t0 + 2 * stride, n_tiles, w);
  }

  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (alone) {
    if (n < a.g) {
      const float inv = 1.f / l;
      const int64_t at = (int64_t)b * a.out_stride + (int64_t)(h * a.g + n) * kDim + 4 * j;
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        store_out2<DT>(a.out, at + 16 * d, o[d][0] * inv, o[d][1] * inv);
        store_out2<DT>(a.out, at + 16 * d + 2, o[d][2] * inv, o[d][3] * inv);
      }
    }
    return;
  }
  // merge the waves
  __syncthreads();
  float* so = reinterpret_cast<float*>(lds);  // [wave][query][128]
  if (n < a.g) {
#pragma unroll
    for (int d = 0; d < 8; ++d)
      *reinterpret_cast<f32x4*>(so + (wave * 16 + n) * kDim + 16 * d + 4 * j) = o[d];
    if (j == 0) {
      // the sums' reference; a wave without a token has none
      sm_m[wave][n] = m == -INFINITY ? -INFINITY : ref;
      sm_l[wave][n] = l;
    }
  }
  __syncthreads();
  for (int i = tid; i < a.g * (kDim / 2); i += 256) {
    const int g = i >> 6, d = (i & 63) * 2;
    float mx = sm_m[0][g];
#pragma unroll
    for (int w = 1; w < 4; ++w) mx = vmax(mx, sm_m[w][g]);
    float L = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      // a wave without a token has -inf, and nothing summed
      const float f = sm_m[w][g] == -INFINITY ? 0.f : fast_exp2(sm_m[w][g] - mx);
      L = fmaf(sm_l[w][g], f, L);
      const float* p = so + (w * 16 + g) * kDim + d;
      o0 = fmaf(p[0], f, o0);
      o1 = fmaf(p[1], f, o1);
    }
    const float inv = 1.f / L;
    const int hq = h * a.g + g;
    if (np == 1) {
      store_out2<DT>(a.out, (int64_t)b * a.out_stride + (int64_t)hq * kDim + d, o0 * inv, o1 * inv);
    } else {
      // (scores of -inf alone: a weight of 0 to be, which NaN would not stand)
      const float f = L == 0.f ? 0.f : inv;
      const int64_t slot = ((int64_t)b * a.hq + hq) * a.n_parts + part;
      *reinterpret_cast<float2*>(a.ws_o + slot * kDim + d) = make_float2(o0 * f, o1 * f);
      if (d == 0) a.ws_lse[slot] = mx + __log2f(L);
    }
  }
}

template <Dt DT> __global__ __launch_bounds__(256) void kv4_reduce_kernel(DecArgs a) {
  const int hq = blockIdx.x, b = blockIdx.y;
  const int ctx = context_len(a, a.lens[b]);
  const int np = parts_of(a, ctx, part_of(a, ctx));
  if (np <= 1) return;
  combine_partitions<DT>(a.ws_o, a.ws_lse, ((int64_t)b * a.hq + hq) * a.n_parts, np, a.out,
                         (int64_t)b * a.out_stride + (int64_t)hq * kDim);
}

// Workgroups that the GPU holds at once: three per CU, fp32 two.
static int round_of(bool fp32) { return fp32 ? 512 : 768; }
// The longest context that is not split.  From 512 (sequence, head) items on whole contexts are
// faster or as fast (us at 8 heads, whole / in 1024, of 1-2k and of 2-4k tokens: 64 sequences
// 24.0 / 29.1 and 43.5 / 44.3, 96 33.3 / 38.9 and 61.0 / 62.2, 128 44.1 / 45.8 and 80.8 / 79.6,
// 192 58.1 / 62.5 and 108 / 114, 256 75.0 / 81.7 and 143 / 150).  The two sides cross below
// that: 32 16.4 / 17.5 and 28.5 / 28.2, 16 16.6 / 16.5 and 28.8 / 20.8, so that up to 63 sequences
// of equal lengths (24.2 / 29.1 and 43.3 / 45.0) are split where whole ones would be faster.
static int32_t whole_context(int64_t items) { return items >= 512 ? 4096 : 768; }

// The longest context that one wave takes, from four rounds of workgroups on (three per
// CU, fp32 two; us, one wave / four: 512 x 1-64 at 8 heads 17.6 / 26.1, 129-256 31.0 /
// 32.5, 2000 x 10-300 93 / 114; fp32 20.0 / 43.0, 37.3 / 49.0, 137 / 191, 256 x 1-256 21.4
// / 25.3).  Below that four waves a head are done sooner: bf16, 256 x 1-256 18.4 / 17.4, 128
// x 1-200 15.4 / 10.6.
static int32_t one_wave_context(int32_t n_seqs, int32_t hkv, bool fp32) {
  return hkv % 4 == 0 && (int64_t)n_seqs * hkv >= 4 * round_of(fp32) ? 4 * kStep : 0;
}

struct Plan {
  int32_t part_tokens, n_parts;
  size_t ws_bytes;
};

static Plan plan(int32_t n_seqs, int32_t hq, int32_t hkv, int32_t block_size, int32_t max_blocks,
                 int32_t max_context_len, int32_t part_tokens, bool fp32) {
  Plan p;
  int64_t cap = std::min<int64_t>((int64_t)max_blocks * block_size, kMaxContext);
  if (max_context_len > 0 && max_context_len < cap) cap = max_context_len;
  if (cap < 1) cap = 1;
  int64_t part = part_tokens;
  if (part <= 0) {
    // Measured on MI355X (us, graph replay).  A workgroup starts and ends in some 4 us, a
    // turn of 256 tokens takes 1.2 of latency, and the second launch 2.5.  So no split
    // up to 768 tokens (32 x 100-600 at 4 heads: 7.8 against 9.5 in 256), nor from 512
    // (sequence, head) items up to 4096 (whole_context).  Else
    // what one round of workgroups (three per CU, fp32 two) makes of the tables, up to
    // 1024 tokens (24 x 100-2063: 768 15.4, 256 17.4, unsplit 17.3; one of 8000: 256
    // 8.4, 768 10.6).  Beyond, contexts of different lengths leave a round's end to a
    // few workgroups: the power of two from a quarter of it on, 1024 to 4096 (200 x 1-6k
    // at one head: 1024 32.9, 2048 36; 16 x 10-30k at 8: 1024 66.9, 2048 67.7, 6144 80;
    // 100 x 2-6k at 4: 1024 45.0, 512 48.6, 4096 63; 64 x 16-32k at 8: 4096 282, 8192 288,
    // 2048 293, 1024 308; 200 x 4-12k at 8: 4096 285, 8192 297, 2048 288).  No more than 64 parts to
    // combine (2 x 60k at 4: 1024 18.3, 768 20.3; one of 115k in fp16: 2048 30.5, 1024
    // 34.8, 4096 34.1).
    const int64_t items = (int64_t)n_seqs * hkv, round = cdiv(cap * items, round_of(fp32));
    part = rounds_part((u32)std::min<int64_t>(round, 1 << 30));
    part = std::max(part, cdiv(cap, 64));
    if (cap <= whole_context(items)) part = cap;
  }
  part = cdiv(std::min(part, cap), kTurn) * kTurn;
  p.part_tokens = (int32_t)part;
  p.n_parts = (int32_t)cdiv(cap, part);
  p.ws_bytes = p.n_parts > 1 ? (size_t)n_seqs * hq * p.n_parts * (kDim + 1) * sizeof(float) : 0;
  return p;
}

template <Dt DT> static void launch(const DecArgs& a, hipStream_t s) {
  // An odd number of partitions: workgroups go round the XCDs and the shader engines of
  // each in turn, so with 4 or 8, of which a captured step sized for the longest context has
  // one or two that hold tokens, those would all fall on one or two engines of four (us,
  // 256 x 300-1,500 in tables of 16,384 tokens at 8 heads 138 and 54, of 8,192 82 and 53,
  // 64 x 500-2,000 in 32,768 53 and 28).  Where every partition holds tokens, the one that
  // is empty costs up to 1% (64 x 16-32k 283 and 285), or nothing (200 x 4-12k 286).
  const dim3 grid(a.c.hkv, a.n_parts | 1, a.n_seqs);
  if (a.c.block_size % kStep == 0)
    hipLaunchKernelGGL((kv4_decode_kernel<DT, true>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((kv4_decode_kernel<DT, false>), grid, dim3(256), 0, s, a);
  if (a.n_parts > 1)
    hipLaunchKernelGGL((kv4_reduce_kernel<DT>), dim3(a.hq, a.n_seqs), dim3(256), 0, s, a);
}

}  // namespace kv4
}  // namespace aac

using namespace aac;

extern "C" size_t aac_kv4_decode_workspace_bytes(int32_t n_seqs, int32_t n_q_heads, int32_t n_kv_heads,
                                                 int32_t head_dim, int32_t block_size,
                                                 int32_t max_blocks_per_seq, int32_t max_context_len,
                                                 int32_t partition_tokens) {
  (void)head_dim;
  if (n_seqs <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || block_size <= 0 || max_blocks_per_seq <= 0)
    return 0;
  // the element type is not known here: the larger of the two plans
  size_t most = 0;
  for (bool fp32 : {false, true})
    most = std::max(most, kv4::plan(n_seqs, n_q_heads, n_kv_heads, block_size, max_blocks_per_seq,
                                    max_context_len, partition_tokens, fp32).ws_bytes);
  return most;
}

extern "C" int aac_kv4_decode(const void* q, int64_t q_seq_stride, const void* k, const void* v,
                              int64_t k_seq_stride, int64_t v_seq_stride, void* cache, int64_t num_blocks,
                              int32_t block_size, const int32_t* block_tables, int32_t max_blocks_per_seq,
                              const int32_t* context_lens, int32_t n_seqs, int32_t max_context_len,
                              int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, float scale, void* out, int64_t out_seq_stride,
                              void* workspace, size_t workspace_bytes, int32_t partition_tokens,
                              int32_t dtype, void* stream) {
  if (n_seqs < 0 || n_q_heads <= 0 || max_blocks_per_seq <= 0 || q_seq_stride < 0 || out_seq_stride < 0)
    return AAC_ERR_INVALID_ARGUMENT;
  if (dtype != AAC_DTYPE_BF16 && dtype != AAC_DTYPE_FP16 && dtype != AAC_DTYPE_FP32)
    return AAC_ERR_UNSUPPORTED;
  if (n_seqs == 0) return AAC_OK;
  const int rc = kv4::check_cache(cache, num_blocks, block_size, n_kv_heads, head_dim);
  if (rc != AAC_OK) return rc;
  if (n_q_heads % n_kv_heads) return AAC_ERR_SHAPE;
  if (n_q_heads / n_kv_heads > 16 || num_blocks > INT32_MAX || n_seqs > 65535) return AAC_ERR_UNSUPPORTED;
  if (!q || !block_tables || !context_lens || !out) return AAC_ERR_INVALID_ARGUMENT;
  const int64_t width = (int64_t)n_q_heads * head_dim;
  if (q_seq_stride < width || out_seq_stride < width) return AAC_ERR_SHAPE;
  const int es = dtype == AAC_DTYPE_FP32 ? 4 : 2;
  if ((uintptr_t)q % 16 || (q_seq_stride * es) % 16 || (uintptr_t)out % 8 || (out_seq_stride * es) % 8)
    return AAC_ERR_MISALIGNED;
  const kv4::Plan p = kv4::plan(n_seqs, n_q_heads, n_kv_heads, block_size, max_blocks_per_seq,
                                max_context_len, partition_tokens, dtype == AAC_DTYPE_FP32);
  if (p.n_parts > 65535) return AAC_ERR_UNSUPPORTED;
  if (p.ws_bytes) {
    if (!workspace || workspace_bytes < p.ws_bytes) return AAC_ERR_WORKSPACE;
    if ((uintptr_t)workspace % 16) return AAC_ERR_MISALIGNED;
  }
  if ((k == nullptr) != (v == nullptr)) return AAC_ERR_INVALID_ARGUMENT;
  if (k) {  // all rows are written before any is read
    const int arc = aac_kv4_append(k, v, k_seq_stride, v_seq_stride, cache, num_blocks, block_size, block_tables,
                                   max_blocks_per_seq, context_lens, n_seqs, n_kv_heads, head_dim, dtype, stream);
    if (arc != AAC_OK) return arc;
  }
  kv4::DecArgs a = {};
  a.q = q;
  a.q_stride = q_seq_stride;
  a.c = {(unsigned char*)cache, num_blocks, block_size, n_kv_heads};
  a.block_tables = block_tables;
  a.max_blocks = max_blocks_per_seq;
  a.lens = context_lens;
  a.lens_add = k ? 1 : 0;
  a.n_seqs = n_seqs;
  a.hq = n_q_heads;
  a.g = n_q_heads / n_kv_heads;
  a.scale_log2 = scale * kLog2e;
  a.out = out;
  a.out_stride = out_seq_stride;
  a.n_parts = p.n_parts;
  a.part_tokens = p.part_tokens;
  // Granlund and Montgomery 1994, Theorem 4.2, for tile numbers below 2^27: magic = floor(2^(27 + l) / d) + 1, l = ceil(log2 d)
  const u32 d = (u32)(block_size / kv4::kTile);
  const int l = d == 1 ? 0 : 32 - __builtin_clz(d - 1);
  a.magic = (uint64_t(1) << (27 + l)) / d + 1;
  a.shift = 27 + l;
  a.alone = kv4::one_wave_context(n_seqs, n_kv_heads, dtype == AAC_DTYPE_FP32);
  if (partition_tokens <= 0 && p.n_parts > 1) {
    const int64_t items = (int64_t)n_seqs * n_kv_heads;
    a.tight = (int32_t)((int64_t)p.n_parts * p.part_tokens / 4);
    a.whole = kv4::whole_context(items);
    a.per_round = (uint64_t)std::min<int64_t>(items, 1 << 15) * 65536 / kv4::round_of(dtype == AAC_DTYPE_FP32);
    a.inv_parts = (u32)(((uint64_t(1) << 32) + p.n_parts - 1) / p.n_parts);
  }
  if (p.ws_bytes) {
    a.ws_o = reinterpret_cast<float*>(workspace);
    a.ws_lse = a.ws_o + (size_t)n_seqs * n_q_heads * p.n_parts * kv4::kDim;
  }
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case AAC_DTYPE_BF16: kv4::launch<Dt::BF16>(a, s); break;
    case AAC_DTYPE_FP16: kv4::launch<Dt::FP16>(a, s); break;
    default: kv4::launch<Dt::FP32>(a, s); break;
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? AAC_OK : (int)e;
}
