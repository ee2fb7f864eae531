// Log probabilities of given tokens, the entropy and the top alternatives of each
// row of logits (gfx950).
//
//   m = max x,  S = sum e^(x - m),  T = sum (x - m) e^(x - m)
//   logp_i = x_i - m - ln S,   entropy = ln S - T / S,
//   the k largest x by (value, lowest index), a NaN counting as larger than every number
//   (the order of aac_argmax_rows).
// T is summed about the maximum, so nothing cancels; an x of -inf adds nothing to S
// or T.  A row with a NaN, with +inf, or of -inf alone has no distribution: NaN, as
// torch.log_softmax gives.
//
// Two launches.  The first streams the logits: a workgroup holds a segment of a row in
// its registers, forms the maximum, then S and T about it, and writes them for each
// wave, and the maximum of each group of 128 neighbouring values (fp32: 64), which
// the 16 lanes of a DPP row hold.  The second, a workgroup a row, joins the sums and
// finds the top k from the group maxima: a value above a bound that k groups reach
// lies in a group that reaches it, so only some k groups of 256 bytes are read again.
// Bound by the read of the logits (bf16, us): 256 x 151,936 16.6 of the first launch and
// 5.4 (top 20) of the second, whose chain of small steps is its cost (cycles of a row's
// workgroup: 2.8k until the sums are there, 1.5k for the bound, 0.9k and 2.9k for the
// groups, 2k for the values, 1.1k for the ranks); 1500 rows 76, 6.0 TB/s (fp32 6.5).
// Tried instead: candidates collected in the first launch, where every wave goes through
// nearly all of its values again (197 against 17); one launch with a workgroup of 16
// waves a row, maxima in LDS (1 row of 151,936, top 20 22.4 against 8.6, 256 rows 26.7
// against 24.4, 300 48 against 30; up to 32,000 columns 5 to 15% faster to 256 rows).
#include <algorithm>
#include <climits>

#include "aac_common.h"

namespace aac {
namespace lp {

typedef unsigned long long u64;

constexpr int kThreads = 256;
constexpr int kChunks = 8;     // 16-byte chunks a thread of the first launch
constexpr int kGroup = 16;     // chunks of a group
constexpr int kMaxTop = 32;
constexpr int kSegChunks = kThreads * kChunks;

struct Args {
  const char* x;
  int64_t stride;  // bytes
  int64_t n_rows;
  int32_t cols, top, n_seg;
  const int64_t* tokens;
  float* logp;
  float* entropy;
  float* top_logp;
  int64_t* top_ids;
  float* ws_sum;  // [n_rows, n_seg * 4 waves, 4]: m, S, T (base 2: sum of 2^d and d 2^d), d of x = m
  float* ws_max;  // [n_rows, n_seg * 128]: group maxima
};

template <Dt DT> struct Row {
  static constexpr int kEs = DT == Dt::FP32 ? 4 : 2;
  static constexpr int kE = 16 / kEs;  // elements of a chunk
  // order_key's low bits carry nothing in a 16-bit type
  static constexpr int kKeyShift = DT == Dt::BF16 ? 16 : DT == Dt::FP16 ? 13 : 0;
  __device__ static float one(const char* p) {
    if constexpr (DT == Dt::FP32) return *reinterpret_cast<const float*>(p);
    else if constexpr (DT == Dt::BF16) return bf16lo(*reinterpret_cast<const u16*>(p));
    else return (float)*reinterpret_cast<const _Float16*>(p);
  }
  __device__ static void unpack(const u32x4& w, float* v) {
    if constexpr (DT == Dt::FP32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(w[e]);
    } else {
      Elem<DT>::unpack8(w, v);
    }
  }
  // Chunk c of a row whose first element is element `mis` of chunk 0; -inf where the
  // chunk lies outside the row.
  __device__ static u32x4 chunk(const char* p, int mis, int cols, int64_t c) {
    const int64_t i0 = c * kE - mis;
    if (i0 >= 0 && i0 + kE <= cols) return *reinterpret_cast<const u32x4*>(p + i0 * kEs);
    constexpr u32 kNone = DT == Dt::BF16 ? 0xff80ff80u : DT == Dt::FP16 ? 0xfc00fc00u : 0xff800000u;
    u32x4 w = {kNone, kNone, kNone, kNone};
    if (i0 < cols) {  // the row's first or last elements
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const int64_t i = i0 + e;
        if (i < 0 || i >= cols) continue;
        if constexpr (DT == Dt::FP32) {
          w[e] = *reinterpret_cast<const u32*>(p + i * 4);
        } else {
          const u32 b = *reinterpret_cast<const u16*>(p + i * 2);
          w[e >> 1] = e & 1 ? (w[e >> 1] & 0xffffu) | b << 16 : (w[e >> 1] & 0xffff0000u) | b;
        }
      }
    }
    return w;
  }
};

// a float's place in the order: NaN largest, -0 as 0
__device__ __forceinline__ u32 order_key(float x) {
  u32 b = __float_as_uint(x);
  if (x != x) return 0xffffffffu;
  if (b == 0x80000000u) b = 0;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// the float of a key whose low `shift` bits were dropped (they are those of the type)
__device__ __forceinline__ float key_float(u32 key, int shift) {
  const u32 b = key << shift;
  return __uint_as_float((b & 0x80000000u ? b ^ 0x80000000u : ~b) >> shift << shift);
}
__device__ __forceinline__ float wave_sum(float x) {
  x = row16_sum(x);
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}

// S and T of one chunk about m, base 2.  The exponent d = x log2 e - m log2 e is one
// fma; the rounding of nm = -m log2 e moves all of them alike and is taken out where the
// sums are joined (`residue`).  An x of -inf has to add 0 to T, so values far below any
// m of this form are raised to a finite one first, two in an instruction in the 16-bit
// types (as unsigned numbers the negative bfloat16 go up with their size); it adds 2^d
// = 0 as before.  Where m is near those values or m log2 e may overflow (FAR), x - m
// comes first.
template <Dt DT> __device__ __forceinline__ bool is_far(float m) {
  return !(m <= 1e36f) || m < (DT == Dt::FP16 ? -6e4f : -1e36f);
}
template <Dt DT, bool FAR>
__device__ __forceinline__ void add_chunk(u32x4 w, float m, float nm, float& S, float& T) {
  typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
  if constexpr (!FAR) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32 x = w[i];  // (a bit cast of a vector's element itself reads its first)
      if constexpr (DT == Dt::BF16)  // at least -9.97e36
        w[i] = __builtin_bit_cast(u32, __builtin_elementwise_min(__builtin_bit_cast(u16x2, x), (u16x2){0xfcf0, 0xfcf0}));
      else if constexpr (DT == Dt::FP16)  // at least -65504
        w[i] = __builtin_bit_cast(u32, __builtin_elementwise_max(__builtin_bit_cast(f16x2, x),
                                                                 (f16x2){(_Float16)-65504.f, (_Float16)-65504.f}));
    }
  }
  float v[Row<DT>::kE];
  Row<DT>::unpack(w, v);
#pragma unroll
  for (int e = 0; e < Row<DT>::kE; ++e) {
    float d;
    if constexpr (FAR) d = (v[e] - m) * kLog2e;
    else d = fmaf(DT == Dt::FP32 ? fmaxf(v[e], -1e37f) : v[e], kLog2e, nm);
    const float p = fast_exp2(d);
    S += p;
    T = fmaf(p, FAR ? fmaxf(d, -1e30f) : d, T);
  }
}
// what d of x = m is, in place of 0
template <Dt DT> __device__ __forceinline__ float residue(float m) {
  return is_far<DT>(m) ? 0.f : fmaf(m, kLog2e, -(m * kLog2e));
}

// Chunks c0, c0 + step, ... of a row, NC of them.  All loads first, from chunks that lie
// within the row (another one's place for those that do not), then the few chunks at
// the row's ends (only where `ends`, the same for the whole wave).
template <Dt DT, int NC>
__device__ __forceinline__ void load_chunks(const char* p, int mis, int cols, int64_t c0, int step, bool ends,
                                            u32x4* w) {
  typedef Row<DT> R;
  const int64_t c_lo = mis ? 1 : 0, c_hi = (cols + mis) / R::kE - 1;  // whole chunks
  if (c_lo <= c_hi) {
#pragma unroll
    for (int u = 0; u < NC; ++u)
      w[u] = __builtin_nontemporal_load(
          reinterpret_cast<const u32x4*>(p + (min(max(c0 + step * u, c_lo), c_hi) * R::kE - mis) * R::kEs));
  }
  if (ends) {
#pragma unroll
    for (int u = 0; u < NC; ++u) {
      const int64_t c = c0 + step * u;
      if (c < c_lo || c > c_hi) w[u] = R::chunk(p, mis, cols, c);
    }
  }
}
// whether any of the n chunks from c on is not whole
template <Dt DT> __device__ __forceinline__ bool has_ends(int mis, int cols, int64_t c, int n) {
  return c < (mis ? 1 : 0) || c + n - 1 > (cols + mis) / Row<DT>::kE - 1;
}

// The maximum over a wave of its chunks (NaN if one is), returned, and those of the
// groups: lane l gets chunk (l >> kOwn) & (NC - 1)'s of its 16 lanes.
// In each step a lane hands half of its values to its partner (lane ^ 15, ^ 7, then ^ 2,
// ^ 1) and keeps the other half, until one is left.
template <int NC> constexpr int kOwn = NC == 8 ? 1 : 2;  // log2 of the lanes that end with one chunk
template <Dt DT, int NC> __device__ __forceinline__ float chunk_maxima(const u32x4* w, int lane, float* group) {
  static_assert(NC == 4 || NC == 8, "two or three halvings");
  constexpr int E = Row<DT>::kE;
  float cm[NC];
#pragma unroll
  for (int u = 0; u < NC; ++u) {
    float v[E];
    Row<DT>::unpack(w[u], v);
    cm[u] = vmax3(v[0], v[1], v[2]);
#pragma unroll
    for (int e = 3; e + 1 < E; e += 2) cm[u] = vmax3(cm[u], v[e], v[e + 1]);
    cm[u] = vmax(cm[u], v[E - 1]);
  }
  const bool b3 = lane & 8, b2 = lane & 4, b1 = lane & 2;
  constexpr int H = NC / 2, Q = NC / 4;
  float h[H], q[Q], g;
#pragma unroll
  for (int i = 0; i < H; ++i) h[i] = vmax(b3 ? cm[i + H] : cm[i], dpp_f<kDppRowMirror>(b3 ? cm[i] : cm[i + H]));
#pragma unroll
  for (int i = 0; i < Q; ++i) q[i] = vmax(b2 ? h[i + Q] : h[i], dpp_f<kDppRowHalfMirror>(b2 ? h[i] : h[i + Q]));
  if constexpr (NC == 8) g = vmax(b1 ? q[1] : q[0], dpp_f<kDppQuadXor2>(b1 ? q[0] : q[1]));
  else g = vmax(q[0], dpp_f<kDppQuadXor2>(q[0]));
  g = vmax(g, dpp_f<kDppQuadXor1>(g));
  *group = g;
  float m = vmax(g, dpp_f<kDppQuadXor2>(g));
  m = vmax(m, dpp_f<kDppRowHalfMirror>(m));
  m = vmax(m, dpp_f<kDppRowMirror>(m));
  m = vmax(m, __shfl_xor(m, 16));
  return vmax(m, __shfl_xor(m, 32));
}

template <Dt DT>
__global__ __launch_bounds__(kThreads, 6) void logprobs_segment_kernel(Args a) {
  typedef Row<DT> R;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.x / a.n_seg;
  const int seg = (int)(blockIdx.x % a.n_seg);
  const char* p = a.x + row * a.stride;
  const int mis = (int)((uintptr_t)p & 15) / R::kEs;
  const int64_t s0 = (int64_t)seg * kSegChunks;
  u32x4 w[kChunks];
  load_chunks<DT, kChunks>(p, mis, a.cols, s0 + tid, kThreads, has_ends<DT>(mis, a.cols, s0, kSegChunks), w);
  float group;
  const float m = chunk_maxima<DT, kChunks>(w, lane, &group);
  if (a.top > 0 && (lane & ((1 << kOwn<kChunks>) - 1)) == 0)
    a.ws_max[(row * a.n_seg + seg) * (kSegChunks / kGroup) +
             ((lane >> kOwn<kChunks>) & (kChunks - 1)) * (kThreads / kGroup) + wave * 4 + (lane >> 4)] = group;
  // The values are unpacked again from here: kept from the maxima they take 64 registers
  // and half of the waves (1500 rows of bf16: 83 against 79 us).
#pragma unroll
  for (int u = 0; u < kChunks; ++u) asm volatile("" : "+v"(w[u]));
  float S = 0.f, T = 0.f;
  if (is_far<DT>(m)) {  // (a NaN or +inf is here, and makes S a NaN; -inf alone adds nothing)
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int u = 0; u < kChunks; ++u) add_chunk<DT, true>(w[u], ref, 0.f, S, T);
  } else {
    const float nm = -(m * kLog2e);
#pragma unroll
    for (int u = 0; u < kChunks; ++u) add_chunk<DT, false>(w[u], m, nm, S, T);
  }
  S = wave_sum(S);
  T = wave_sum(T);
  if (lane == 0)
    *reinterpret_cast<f32x4*>(a.ws_sum + ((row * a.n_seg + seg) * 4 + wave) * 4) =
        f32x4{m, S, T, residue<DT>(m)};
}

template <int CTRL> __device__ __forceinline__ u32 dpp_u(u32 x) {
  return (u32)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false);
}
// The smallest and the largest key of the wave.
__device__ __forceinline__ uint2 wave_range(u32 key) {
  u32 lo = key, hi = key;
#define AAC_STEP(c) lo = min(lo, dpp_u<c>(lo)), hi = max(hi, dpp_u<c>(hi))
  AAC_STEP(kDppQuadXor1);
  AAC_STEP(kDppQuadXor2);
  AAC_STEP(kDppRowHalfMirror);
  AAC_STEP(kDppRowMirror);
#undef AAC_STEP
  u32 l = 0xffffffffu, h = 0;
#pragma unroll
  for (int r = 0; r < 64; r += 16) {
    l = min(l, (u32)__builtin_amdgcn_readlane((int)lo, r));
    h = max(h, (u32)__builtin_amdgcn_readlane((int)hi, r));
  }
  return make_uint2(l, h);
}

// The wave's k-th and j-th largest of 64 keys, bit by bit from the first in which the keys
// differ; near: down to a 16th of the way from there to the largest key, the rest left
// at 0, so that the result is at most that key.  A step takes some 130 cycles, of counts
// that only the scalar unit takes (two bits a step cost more: three counts for each key's
// two bits).
__device__ __forceinline__ uint2 kth_of_wave(u32 key, int k, int j, bool near) {
  const uint2 range = wave_range(key);
  if (k == 1) return make_uint2(range.y, range.y);
  const int top = 32 - __builtin_clz(range.x ^ range.y | 1u);  // bits from here up are alike
  u32 tk = top < 32 ? range.y >> top << top : 0, tj = tk;
#pragma unroll 1
  for (int s = top - 1; s >= 0; --s) {
    const u32 bit = 1u << s;
    if ((int)__popcll(__ballot(key >= (tk | bit))) >= k) tk |= bit;
    if ((int)__popcll(__ballot(key >= (tj | bit))) >= j) tj |= bit;
    if (near && (range.y - tk) >> s >= 16) break;
  }
  return make_uint2(tk, tj);
}

__device__ __forceinline__ u32 lanes_below(unsigned long long mask) {
  return __builtin_amdgcn_mbcnt_hi((u32)(mask >> 32), __builtin_amdgcn_mbcnt_lo((u32)mask, 0u));
}

// A candidate as one number: larger for the larger value, then for the lower index.
__device__ __forceinline__ u64 entry(u32 key, u32 index) { return (u64)key << 32 | (u32)~index; }
__device__ __forceinline__ u32 index_of(u64 e) { return ~(u32)e; }

// Hands each of the list's n entries that is among the k largest to put(rank, entry).
// Four lanes an entry, each against eight entries at a time, so that the reads overlap:
// entries n to the next multiple of 32 are set to 0 first, which is below every entry.
constexpr int kListPad = 32;
template <typename F> __device__ __forceinline__ void ranked(u64* list, int n, int k, F put) {
  if ((int)threadIdx.x < kListPad) list[n + threadIdx.x] = 0;
  __syncthreads();
  const int part = threadIdx.x & 3;
  for (int i = threadIdx.x >> 2; i < n; i += kThreads / 4) {
    const u64 c = list[i];
    int rank = 0;
    for (int j = 0; j < n; j += kListPad) {
#pragma unroll
      for (int z = 0; z < 8; ++z) rank += list[j + 8 * part + z] > c;
    }
    rank += __builtin_amdgcn_update_dpp(0, rank, kDppQuadXor1, 0xF, 0xF, false);
    rank += __builtin_amdgcn_update_dpp(0, rank, kDppQuadXor2, 0xF, 0xF, false);
    if (part == 0 && rank < k) put(rank, c);
  }
}

// Entries a list has to hold in the ordered search: in each of the four waves fewer than k
// lanes have a key above the bound, `per` entries each, and k entries equal to it are kept.
__host__ __device__ inline int list_cap(int k, int per) { return 4 * ((k - 1) * per + k) + kListPad; }
constexpr int kFast = 512;      // entries the list holds in the plain search
constexpr int kFastGroups = 128;  // groups it takes, 64 at a time
constexpr int kHeld = 6;  // group maxima a thread keeps

// (m, S, T) of one part of a row, joined with others' about the row's m.  r: d of x = m.
struct Sums {
  float m = -INFINITY, S = 0.f, T = 0.f;
};
__device__ __forceinline__ void join(Sums& row, const f32x4& part) {
  // (a part of -inf alone has S = T = 0)
  const float d = fmaxf((part[0] - row.m) * kLog2e, -1e30f) - part[3], f = fast_exp2(d);
  row.S = fmaf(part[1], f, row.S);
  row.T += f * fmaf(d, part[1], part[2]);
}

// The log of a row's sum, NaN where there is no distribution; writes the entropy and the
// token's log probability (one thread).
template <Dt DT>
__device__ __forceinline__ float finish_sums(const Args& a, int64_t row, const Sums& s, int64_t token, float xt) {
  const bool fine = fabsf(s.m) < INFINITY && s.S == s.S;
  const float log_s = fine ? logf(s.S) : __uint_as_float(0x7fc00000u);
  if (threadIdx.x == 0) {
    a.entropy[row] = log_s - s.T / s.S * 0.6931471805599453f;
    a.logp[row] = token < 0 ? 0.f : token < a.cols ? xt - s.m - log_s : __uint_as_float(0x7fc00000u);
  }
  return log_s;
}

// The top k of a row from its group maxima, by a workgroup of four waves.  own: those
// of groups threadIdx.x + 256 i.
template <Dt DT>
__device__ __forceinline__ void write_top(const Args& a, int64_t row, const Sums& sums, float log_s,
                                          const float* gmax, const float* own, int n_groups, u64* list) {
  typedef Row<DT> R;
  constexpr int E = R::kE, kShift = R::kKeyShift;
  __shared__ uint2 s_tau[4];
  __shared__ u32 s_n[4];
  __shared__ u32 s_group[kMaxTop], s_sorted[kMaxTop], s_list[kFastGroups];
  __shared__ u64 s_best[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const char* x = a.x + row * a.stride;
  const int k = a.top;
  float* top_logp = a.top_logp + row * k;
  int64_t* top_ids = a.top_ids + row * k;
  auto key_of = [](float v) { return order_key(v) >> kShift; };
  auto put = [&](int r, u64 c) {
    top_logp[r] = key_float((u32)(c >> 32), kShift) - sums.m - log_s;
    top_ids[r] = index_of(c);
  };

  if (!(sums.S == sums.S) || sums.m == INFINITY) {
    // a NaN or +inf somewhere: k selections over the row, by value and index
    u64 last = ~(u64)0;
    for (int r = 0; r < k; ++r) {
      u64 best = 0;
      for (int i = tid; i < a.cols; i += kThreads) {
        const u64 e = entry(order_key(R::one(x + (int64_t)i * R::kEs)), (u32)i);
        if ((r == 0 || e < last) && e > best) best = e;
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        const u64 other = (u64)__shfl_xor((u32)(best >> 32), o) << 32 | (u32)__shfl_xor((u32)best, o);
        best = max(best, other);
      }
      if (lane == 0) s_best[wave] = best;
      __syncthreads();
      for (int q = 0; q < 4; ++q) best = max(best, s_best[q]);
      last = best;
      if (tid == 0) {
        top_logp[r] = __uint_as_float(0x7fc00000u);
        top_ids[r] = index_of(best);
      }
      __syncthreads();
    }
    return;
  }

  if (tid < 4) s_n[tid] = 0;
  u32 held[kHeld], best = 0;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    held[i] = tid + i * kThreads < n_groups ? key_of(own[i]) : 0;
    best = max(best, held[i]);
  }
  for (int g = tid + kHeld * kThreads; g < n_groups; g += kThreads) best = max(best, key_of(gmax[g]));

  // A bound of the row's k-th largest from the lanes' best keys: in a wave the k-th
  // largest has k entries at or above it, so the largest of the waves' holds; and so does
  // the smallest of the (k / n)-th largest of n waves, which lies higher for values in no
  // order (top 20 of four waves: some 30 of 256 lanes are above it, not 80).  The first
  // keeps the lists short whatever the order.
  auto bound = [&](u32 key, int n, bool near) {
    const uint2 t = kth_of_wave(key, k, (k + n - 1) / n, near);
    if (lane == 0) s_tau[wave] = t;
    __syncthreads();
    u32 hi = 0, lo = 0xffffffffu;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      hi = max(hi, s_tau[q].x);
      if (q < n) lo = min(lo, s_tau[q].y);
    }
    return max(hi, lo);
  };

  // Plain search: a bound, every group that reaches it, every value of those that reaches
  // it, their ranks.  Some 1.5 k groups and 2 k values of a row in no order.  A row of few
  // groups is read whole, and the bound comes from the lanes' values: of some k groups
  // the k-th largest maximum says little.  (256 rows, us against the ordered search below:
  // 2,048 columns top 20 10.0 and 14.2; 32,000, where more than 64 groups are listed in
  // some row, top 32 13.8 and 17.9.)
  constexpr int kRound = 64;
  const int mis = (int)((uintptr_t)x & 15) / R::kEs;
  const int in_row = (a.cols + mis + kGroup * E - 1) / (kGroup * E);
  const bool few = in_row <= kRound;
  // A bit for each hit, one atomic a lane and a loop over its bits: a branch for each
  // value would cost most of what the row's workgroup takes.  (The counter's address as
  // one that may differ between lanes: of one that does not, the compiler adds up the
  // lanes' counts itself, lane after lane.)
  int zero = 0;
  asm volatile("" : "+v"(zero));
  u32 tau = 0;
  if (!few) {
    tau = bound(best, min(4, n_groups / 64), true);
    u32 hits = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) hits |= held[i] >= tau ? 1u << i : 0u;
    if (hits) {
      u32 at = atomicAdd(&s_n[zero], (u32)__popc(hits));
      for (; hits && at < (u32)kFastGroups; hits &= hits - 1) s_list[at++] = tid + (__ffs(hits) - 1) * kThreads;
    }
    for (int g = tid + kHeld * kThreads; g < n_groups; g += kThreads) {
      if (key_of(gmax[g]) < tau) continue;
      const u32 at = atomicAdd(&s_n[0], 1u);
      if (at < (u32)kFastGroups) s_list[at] = g;
    }
  } else if (tid < in_row) {
    s_list[tid] = tid;
  }
  __syncthreads();
  const u32 n_listed = few ? in_row : s_n[0];
  if (n_listed <= (u32)kFastGroups) {
    constexpr int kFastPer = kRound * kGroup / kThreads;
#pragma unroll 1
    for (u32 g0 = 0; g0 < n_listed; g0 += kRound) {
      u32x4 w[kFastPer];
      int i0[kFastPer];
#pragma unroll
      for (int q = 0; q < kFastPer; ++q) {
        const u32 c = tid + q * kThreads;
        i0[q] = INT_MAX;
        if (g0 + c / kGroup < n_listed) {
          const int ch = (int)s_list[g0 + c / kGroup] * kGroup + c % kGroup;
          i0[q] = ch * E - mis;
          w[q] = R::chunk(x, mis, a.cols, ch);
        }
      }
      if (few) {
        u32 mine = 0;
#pragma unroll
        for (int q = 0; q < kFastPer; ++q) {
          if (i0[q] == INT_MAX) continue;
          float v[E];
          R::unpack(w[q], v);
          float m = v[0];
#pragma unroll
          for (int e = 1; e < E; ++e) m = fmaxf(m, v[e]);
          mine = max(mine, key_of(m));
        }
        tau = bound(mine, min(4, max(1, in_row * kGroup / 64)), true);
      }
      // (as floats: there is no NaN, and -0 is not below 0)
      const u32 none = key_of(-INFINITY);
      const float least = tau <= none ? -INFINITY : key_float(tau, kShift);
      static_assert(kFastPer * E <= 32, "a bit for each value");
      u32 hit = 0;
#pragma unroll
      for (int q = 0; q < kFastPer; ++q) {
        if (g0 + q * (kThreads / kGroup) >= n_listed) break;  // workgroup-uniform
        float v[E];
        R::unpack(w[q], v);
        u32 in = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) in |= v[e] >= least ? 1u << e : 0u;
        // (what lies outside the row, and where no chunk was read, is not in)
        const int lo = max(-i0[q], 0), hi = min(a.cols - i0[q], E);
        hit |= (hi <= 0 ? 0u : in & ((1u << hi) - 1u) & ~((1u << lo) - 1u)) << (q * E);
      }
      if (hit) {
        u32 at = atomicAdd(&s_n[zero + 1], (u32)__popc(hit));
        for (; hit && at < (u32)kFast; hit &= hit - 1) {
          const int bit = __ffs(hit) - 1, q = bit / E, d = bit % E * R::kEs / 4;
          u32 pair = 0;
          int i = 0;
#pragma unroll
          for (int y = 0; y < kFastPer; ++y) {
            const u32 x01 = d & 1 ? w[y][1] : w[y][0], x23 = d & 1 ? w[y][3] : w[y][2];
            pair = q == y ? (d & 2 ? x23 : x01) : pair;
            i = q == y ? i0[y] : i;
          }
          float v;
          if constexpr (DT == Dt::FP32) v = __uint_as_float(pair);
          else if constexpr (DT == Dt::BF16) v = bit & 1 ? bf16hi(pair) : bf16lo(pair);
          else v = bit & 1 ? f16hi(pair) : f16lo(pair);
          list[at++] = entry(key_of(v), (u32)(i + bit % E));
        }
      }
    }
    __syncthreads();
    const int n = (int)s_n[1];
    if (n <= kFast) {
      ranked(list, n, k, put);
      return;
    }
  }

  // Ordered search, for rows with many equal values (a mask of -inf) or values in order:
  // exact bounds, and of the entries equal to a bound only the first k of each wave.
  __syncthreads();
  tau = bound(best, min(4, n_groups / 64), false);
  // This wave's entries above the bound go to the list in any order, of those equal to it
  // the first k in index order (group g0 + lane, g0 rising).
  auto each_group = [&](auto f) {
    for (int g0 = wave * 64, i = 0; g0 < n_groups; g0 += kThreads, ++i) {
      const int g = g0 + lane;
      u32 key = 0;
#pragma unroll
      for (int z = 0; z < kHeld; ++z) key = i == z ? held[z] : key;
      if (i >= kHeld && g < n_groups) key = key_of(gmax[g]);
      f(key, (u32)g);
    }
  };
  u32 above = 0, ties = 0;
  each_group([&](u32 key, u32) {
    above += (u32)__popcll(__ballot(key > tau));
    ties += (u32)__popcll(__ballot(key == tau));
  });
  u32 at = 0;
  if (lane == 0) at = atomicAdd(&s_n[2], above + min(ties, (u32)k));
  at = __builtin_amdgcn_readfirstlane(at);
  u32 tie_at = at + above;
  const u32 tie_end = tie_at + min(ties, (u32)k);
  each_group([&](u32 key, u32 g) {
    const unsigned long long gt = __ballot(key > tau), eq = __ballot(key == tau);
    const u32 pos = key > tau ? at + lanes_below(gt) : tie_at + lanes_below(eq);
    if (key > tau || (key == tau && pos < tie_end)) list[pos] = entry(key, g);
    at += (u32)__popcll(gt);
    tie_at += (u32)__popcll(eq);
  });
  if (tid < kMaxTop) s_group[tid] = 0xffffffffu;
  __syncthreads();
  ranked(list, (int)s_n[2], k, [&](int r, u64 c) { s_group[r] = index_of(c); });
  __syncthreads();
  // the k groups in index order, so that their values' lanes are in index order too
  if (tid < k) {
    int r = 0;
#pragma unroll
    for (int j = 0; j < kMaxTop; ++j) r += s_group[j] < s_group[tid];
    s_sorted[r] = s_group[tid];
  }
  __syncthreads();

  constexpr int kPer = kMaxTop * kGroup / kThreads;  // chunks a thread
  u32x4 w[kPer];
  int64_t i0[kPer];
  best = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int c = tid + q * kThreads;  // a wave's chunks: groups in order
    i0[q] = INT_MAX;
    if (c < k * kGroup) {
      const int64_t ch = (int64_t)s_sorted[c / kGroup] * kGroup + c % kGroup;
      w[q] = R::chunk(x, mis, a.cols, ch);
      i0[q] = ch * E - mis;
      float v[E];
      R::unpack(w[q], v);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i0[q] + e >= 0 && i0[q] + e < a.cols) best = max(best, key_of(v[e]));
    }
  }
  tau = bound(best, min(4, (k * kGroup + 63) / 64), false);
  // Per lane: values above the bound (11 bits), ties in each of the two chunks (10 bits
  // each, of at most 8 x 64); one scan over the wave gives every lane its places.
  static_assert(kPer <= 2, "two counts of ties");
  u32 key[kPer][E], count = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    float v[E];
    R::unpack(w[q], v);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool in = i0[q] + e >= 0 && i0[q] + e < a.cols;
      key[q][e] = in ? key_of(v[e]) : 0;
      count += key[q][e] > tau ? 1u : 0u;
      count += in && key[q][e] == tau ? 1u << (11 + 10 * q) : 0u;
    }
  }
  u32 incl = count;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u32 t = __shfl_up(incl, o);
    if (lane >= o) incl += t;
  }
  const u32 all = __builtin_amdgcn_readlane(incl, 63), mine = incl - count;
  above = all & 0x7ffu;
  ties = min((all >> 11 & 0x3ffu) + (all >> 21), (u32)k);
  at = 0;
  if (lane == 0) at = atomicAdd(&s_n[3], above + ties);
  at = __builtin_amdgcn_readfirstlane(at);
  u32 pos = at + (mine & 0x7ffu);
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    u32 tie = q == 0 ? mine >> 11 & 0x3ffu : (all >> 11 & 0x3ffu) + (mine >> 21);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool in = i0[q] + e >= 0 && i0[q] + e < a.cols;
      if (key[q][e] > tau) list[pos++] = entry(key[q][e], (u32)(i0[q] + e));
      if (in && key[q][e] == tau) {
        if (tie < ties) list[at + above + tie] = entry(key[q][e], (u32)(i0[q] + e));
        ++tie;
      }
    }
  }
  __syncthreads();
  ranked(list, (int)s_n[3], k, put);
}

template <Dt DT>
__global__ __launch_bounds__(kThreads) void logprobs_merge_kernel(Args a) {
  typedef Row<DT> R;
  extern __shared__ u64 list[];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int n_groups = a.n_seg * (kSegChunks / kGroup);
  const int64_t token = a.tokens[row];
  // All that the row's chain of steps starts from is asked for at once.
  const float* gmax = a.ws_max + row * n_groups;
  float own[kHeld];
  if (a.top > 0) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) own[i] = gmax[min((int)threadIdx.x + i * kThreads, n_groups - 1)];
  }
  // every wave joins the sums for itself
  const f32x4* parts = reinterpret_cast<const f32x4*>(a.ws_sum) + row * a.n_seg * 4;
  const int n_parts = a.n_seg * 4;
  f32x4 first = parts[min(lane, n_parts - 1)];
  const float xt = R::one(a.x + row * a.stride + (token >= 0 && token < a.cols ? token : 0) * R::kEs);
  if (lane >= n_parts) first = f32x4{-INFINITY, 0.f, 0.f, 0.f};
  Sums s;
  s.m = first[0];
  for (int i = lane + 64; i < n_parts; i += 64) s.m = fmaxf(s.m, parts[i][0]);
  s.m = wave_max(s.m);
  join(s, first);
  for (int i = lane + 64; i < n_parts; i += 64) join(s, parts[i]);
  s.S = wave_sum(s.S);
  s.T = wave_sum(s.T);
  const float log_s = finish_sums<DT>(a, row, s, token, xt);
  if (a.top > 0) write_top<DT>(a, row, s, log_s, gmax, own, n_groups, list);
}

static int seg_of(int64_t cols, int es) {
  const int e = 16 / es;
  // the row may start anywhere within its first chunk
  return (int)cdiv(cols + 2 * (e - 1), (int64_t)e * kSegChunks);
}

template <Dt DT> static void launch(const Args& a, hipStream_t s) {
  // group maxima a lane of the second launch goes through, or its chunks' elements
  const int per = std::max(a.n_seg * (kSegChunks / kGroup) / kThreads + 1,
                           kMaxTop * kGroup / kThreads * Row<DT>::kE);
  const size_t lds = a.top ? (size_t)std::max(list_cap(a.top, per), kFast + kListPad) * sizeof(u64) : 0;
  hipLaunchKernelGGL((logprobs_segment_kernel<DT>), dim3((unsigned)(a.n_rows * a.n_seg)), dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL((logprobs_merge_kernel<DT>), dim3((unsigned)a.n_rows), dim3(kThreads), lds, s, a);
}

}  // namespace lp
}  // namespace aac

using namespace aac;

extern "C" size_t aac_logprobs_workspace_bytes(int64_t n_rows, int64_t n_cols, int32_t top_k) {
  if (n_rows <= 0 || n_cols <= 0 || top_k < 0) return 0;
  // fp32 rows have the most segments
  const size_t segs = (size_t)n_rows * lp::seg_of(n_cols, 4);
  return segs * 64 + (top_k ? segs * (lp::kThreads / lp::kGroup * lp::kChunks) * 4 : 0);
}

extern "C" int aac_token_logprobs(const void* logits, int64_t row_stride, int64_t n_rows, int64_t n_cols,
                                  const int64_t* tokens, int32_t top_k, float* logprobs, float* entropy,
                                  float* top_logprobs, int64_t* top_ids, void* workspace,
                                  size_t workspace_bytes, int32_t dtype, void* stream) {
  if (dtype != AAC_DTYPE_BF16 && dtype != AAC_DTYPE_FP16 && dtype != AAC_DTYPE_FP32)
    return AAC_ERR_UNSUPPORTED;
  if (n_rows < 0 || n_cols <= 0 || top_k < 0 || row_stride < n_cols) return AAC_ERR_INVALID_ARGUMENT;
  if (top_k > lp::kMaxTop || n_cols > AAC_LOGPROBS_MAX_COLS) return AAC_ERR_UNSUPPORTED;
  if (top_k > n_cols) return AAC_ERR_SHAPE;
  if (n_rows == 0) return AAC_OK;
  if (!logits || !tokens || !logprobs || !entropy || (top_k && (!top_logprobs || !top_ids)))
    return AAC_ERR_INVALID_ARGUMENT;
  const int es = dtype == AAC_DTYPE_FP32 ? 4 : 2;
  if ((uintptr_t)logits % es) return AAC_ERR_MISALIGNED;
  if (!workspace || workspace_bytes < aac_logprobs_workspace_bytes(n_rows, n_cols, top_k))
    return AAC_ERR_WORKSPACE;
  if ((uintptr_t)workspace % 16) return AAC_ERR_MISALIGNED;
  lp::Args a = {};
  a.x = (const char*)logits;
  a.stride = row_stride * es;
  a.n_rows = n_rows;
  a.cols = (int32_t)n_cols;
  a.top = top_k;
  a.n_seg = lp::seg_of(n_cols, es);
  if (n_rows * a.n_seg >= (1 << 24)) return AAC_ERR_UNSUPPORTED;  // (a launch numbers its threads in 32 bits)
  a.tokens = tokens;
  a.logp = logprobs;
  a.entropy = entropy;
  a.top_logp = top_logprobs;
  a.top_ids = top_ids;
  a.ws_sum = (float*)workspace;
  a.ws_max = (float*)((char*)workspace + (size_t)n_rows * a.n_seg * 64);
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case AAC_DTYPE_BF16: lp::launch<Dt::BF16>(a, s); break;
    case AAC_DTYPE_FP16: lp::launch<Dt::FP16>(a, s); break;
    default: lp::launch<Dt::FP32>(a, s); break;
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? AAC_OK : (int)e;
}
