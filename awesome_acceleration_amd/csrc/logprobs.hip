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
// finds the top k from the group maxima: with groups ordered by (maximum, lowest
// index), a value outside the first k groups has k better ones, so only those k
// groups, k x 256 bytes, are read again.  (Collecting candidates in the first
// launch instead, from a bound of each segment, had every wave go through nearly all
// of its values a second time: 197 us against the 17 of the read at 256 x 151,936.)
// Bound by the read of the logits.
#include <algorithm>
#include <climits>

#include "aac_common.h"

namespace aac {
namespace lp {

constexpr int kThreads = 256;
constexpr int kChunks = 8;     // 16-byte chunks a thread of the first launch
constexpr int kGroup = 16;     // chunks of a group
constexpr int kMaxTop = 32;

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
  float* ws_sum;  // [n_rows, n_seg * 4 waves, 4]: m, S, T (base 2: sum of 2^d and d 2^d)
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
// candidate order: larger value first, then lower index
__device__ __forceinline__ bool before(u32 ka, u32 ia, u32 kb, u32 ib) {
  return ka > kb || (ka == kb && ia < ib);
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
// sums are joined (`residue`).  Where m log2 e may overflow (and for -inf) x - m comes
// first.
template <Dt DT, bool FAR>
__device__ __forceinline__ void add_chunk(const u32x4& w, float m, float nm, float& S, float& T) {
  float v[Row<DT>::kE];
  Row<DT>::unpack(w, v);
#pragma unroll
  for (int e = 0; e < Row<DT>::kE; ++e) {
    const float d = FAR ? (v[e] - m) * kLog2e : fmaf(v[e], kLog2e, nm);
    const float p = fast_exp2(d);
    S += p;
    T = fmaf(p, fmaxf(d, -1e30f), T);  // (d = -inf: adds 0; a NaN stays in S)
  }
}
__device__ __forceinline__ bool is_far(float m) { return !(fabsf(m) <= 1e38f); }
// what d of x = m is, in place of 0
__device__ __forceinline__ float residue(float m) {
  return is_far(m) ? 0.f : fmaf(m, kLog2e, -(m * kLog2e));
}

template <Dt DT>
__global__ __launch_bounds__(kThreads) void logprobs_segment_kernel(Args a) {
  typedef Row<DT> R;
  constexpr int E = R::kE;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.x / a.n_seg;
  const int seg = (int)(blockIdx.x % a.n_seg);
  const char* p = a.x + row * a.stride;
  const int mis = (int)((uintptr_t)p & 15) / R::kEs;
  const int64_t c0 = (int64_t)seg * (kThreads * kChunks) + tid;  // chunk c0 + 256 u

  u32x4 w[kChunks];
#pragma unroll
  for (int u = 0; u < kChunks; ++u) w[u] = R::chunk(p, mis, a.cols, c0 + kThreads * u);

  float gm[kChunks], m = -INFINITY;
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    float v[E];
    R::unpack(w[u], v);
    gm[u] = v[0];
#pragma unroll
    for (int e = 1; e < E; ++e) gm[u] = fmaxf(gm[u], v[e]);
    gm[u] = row16_max(gm[u]);
    m = fmaxf(m, gm[u]);
  }
  m = fmaxf(m, __shfl_xor(m, 16));
  m = fmaxf(m, __shfl_xor(m, 32));
  if (a.top > 0) {  // lane u of each 16 writes the maximum of chunk u's group
    float g = gm[0];
#pragma unroll
    for (int u = 1; u < kChunks; ++u) g = (lane & 15) == u ? gm[u] : g;
    if ((lane & 15) < kChunks)
      a.ws_max[(row * a.n_seg + seg) * (kThreads / kGroup * kChunks) + (lane & 15) * (kThreads / kGroup) +
               wave * 4 + (lane >> 4)] = g;
  }

  float S = 0.f, T = 0.f;
  if (is_far(m)) {
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll 1
    for (int u = 0; u < kChunks; ++u) add_chunk<DT, true>(w[u], ref, 0.f, S, T);
  } else {
    const float nm = -(m * kLog2e);
#pragma unroll
    for (int u = 0; u < kChunks; ++u) add_chunk<DT, false>(w[u], m, nm, S, T);
  }
  S = wave_sum(S);
  T = wave_sum(T);
  if (lane == 0)
    *reinterpret_cast<f32x4*>(a.ws_sum + ((row * a.n_seg + seg) * 4 + wave) * 4) = f32x4{m, S, T, 0.f};
}

// The wave's k-th largest of 64 keys (0 if it has fewer above 0), bit by bit.
__device__ __forceinline__ u32 kth_of_wave(u32 key, int k, int bits) {
  u32 tau = 0;
#pragma unroll 1
  for (u32 bit = 1u << (bits - 1); bit; bit >>= 1)
    if ((int)__popcll(__ballot(key >= (tau | bit))) >= k) tau |= bit;
  return tau;
}

// rank[i] of the list's n entries, handed to put(rank, entry) for the first k
template <typename F>
__device__ __forceinline__ void ranked(const uint2* list, int n, int k, F put) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint2 c = list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += before(list[j].x, list[j].y, c.x, c.y);
    if (rank < k) put(rank, c);
  }
}

// Entries (key, index) a list has to hold: in each of the four waves fewer than k lanes
// have a key above the bound, `per` entries each, and k entries equal to it are kept.
__host__ __device__ inline int list_cap(int k, int per) { return 4 * ((k - 1) * per + k); }

template <Dt DT>
__global__ __launch_bounds__(kThreads) void logprobs_merge_kernel(Args a) {
  typedef Row<DT> R;
  constexpr int E = R::kE, kShift = R::kKeyShift, kBits = 32 - kShift;
  extern __shared__ uint2 list[];
  __shared__ u32 s_tau[4], s_n[2];
  __shared__ u32 s_group[kMaxTop], s_sorted[kMaxTop];
  __shared__ uint2 s_best[4];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const char* x = a.x + row * a.stride;
  const int n_groups = a.n_seg * (kThreads / kGroup * kChunks);
  const float* gmax = a.ws_max + row * n_groups;
  const int64_t token = a.tokens[row];
  const bool real = token >= 0 && token < a.cols;
  const float xt = R::one(x + (real ? token : 0) * R::kEs);
  if (tid < 2) s_n[tid] = 0;

  // every wave joins the sums for itself
  const f32x4* sums = reinterpret_cast<const f32x4*>(a.ws_sum) + row * a.n_seg * 4;
  float m = -INFINITY, S = 0.f, T = 0.f;
  for (int s = lane; s < a.n_seg * 4; s += 64) m = fmaxf(m, sums[s][0]);
  m = wave_max(m);
  for (int s = lane; s < a.n_seg * 4; s += 64) {
    const f32x4 v = sums[s];
    const float r = residue(v[0]);
    // (a wave of -inf alone has S = T = 0)
    const float d = fmaxf((v[0] - m) * kLog2e, -1e30f), f = fast_exp2(d - r);
    S = fmaf(v[1], f, S);
    T += f * fmaf(d - r, v[1], v[2]);
  }
  S = wave_sum(S);
  T = wave_sum(T);
  const bool fine = fabsf(m) < INFINITY && S == S;
  const float log_s = fine ? logf(S) : __uint_as_float(0x7fc00000u);
  if (tid == 0) {
    a.entropy[row] = log_s - T / S * 0.6931471805599453f;
    a.logp[row] = real ? xt - m - log_s : token < 0 ? 0.f : __uint_as_float(0x7fc00000u);
  }
  if (a.top == 0) return;
  float* top_logp = a.top_logp + row * a.top;
  int64_t* top_ids = a.top_ids + row * a.top;

  if (!fine && !(m == -INFINITY && S == S)) {
    // a NaN or +inf somewhere: k selections over the row, by value and index
    u32 lk = 0xffffffffu, li = 0;
    for (int r = 0; r < a.top; ++r) {
      u32 bk = 0, bi = 0xffffffffu;
      for (int i = tid; i < a.cols; i += kThreads) {
        const u32 key = order_key(R::one(x + (int64_t)i * R::kEs));
        if ((r == 0 || before(lk, li, key, (u32)i)) && before(key, (u32)i, bk, bi)) {
          bk = key;
          bi = (u32)i;
        }
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        const u32 ok = __shfl_xor(bk, o), oi = __shfl_xor(bi, o);
        if (before(ok, oi, bk, bi)) {
          bk = ok;
          bi = oi;
        }
      }
      if (lane == 0) s_best[wave] = make_uint2(bk, bi);
      __syncthreads();
      uint2 best = s_best[0];
      for (int q = 1; q < 4; ++q)
        if (before(s_best[q].x, s_best[q].y, best.x, best.y)) best = s_best[q];
      lk = best.x;
      li = best.y;
      if (tid == 0) {
        top_logp[r] = __uint_as_float(0x7fc00000u);
        top_ids[r] = li;
      }
      __syncthreads();
    }
    return;
  }

  // In a wave, the k-th largest of the lanes' best keys has k entries at or above it; the
  // largest such bound of the four waves bounds the row's k-th.
  const int k = a.top;
  auto bound = [&](u32 best) {
    const u32 t = kth_of_wave(best, k, kBits);
    if (lane == 0) s_tau[wave] = t;
    __syncthreads();
    return max(max(s_tau[0], s_tau[1]), max(s_tau[2], s_tau[3]));
  };
  u32 best = 0;
  for (int g = tid; g < n_groups; g += kThreads) best = max(best, order_key(gmax[g]) >> kShift);
  u32 tau = bound(best);
  u32 ties = 0;  // of this wave, in index order
  for (int g0 = wave * 64; g0 < n_groups; g0 += kThreads) {
    const int g = g0 + lane;
    const u32 key = g < n_groups ? order_key(gmax[g]) >> kShift : 0;
    if (g < n_groups && key > tau) list[atomicAdd(&s_n[0], 1u)] = make_uint2(key, g);
    const unsigned long long eq = __ballot(g < n_groups && key == tau);
    const u32 at = ties + __builtin_amdgcn_mbcnt_hi((u32)(eq >> 32), __builtin_amdgcn_mbcnt_lo((u32)eq, 0u));
    if (g < n_groups && key == tau && at < (u32)k) list[atomicAdd(&s_n[0], 1u)] = make_uint2(key, g);
    ties += (u32)__popcll(eq);
  }
  __syncthreads();
  if (tid < kMaxTop) s_group[tid] = 0xffffffffu;
  __syncthreads();
  ranked(list, (int)s_n[0], k, [&](int r, uint2 c) { s_group[r] = c.y; });
  __syncthreads();
  // the k groups in index order, so that their values' lanes are in index order too
  if (tid < k) {
    int r = 0;
    for (int j = 0; j < k; ++j) r += s_group[j] < s_group[tid] || (s_group[j] == s_group[tid] && j < tid);
    s_sorted[r] = s_group[tid];
  }
  __syncthreads();

  const int mis = (int)((uintptr_t)x & 15) / R::kEs;
  constexpr int kPer = kMaxTop * kGroup / kThreads;  // chunks a thread
  u32x4 w[kPer];
  int64_t i0[kPer];
  best = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int c = tid + q * kThreads;  // a wave's chunks: groups in order
    i0[q] = INT_MAX;
    if (c < k * kGroup && s_sorted[c / kGroup] != 0xffffffffu) {
      const int64_t ch = (int64_t)s_sorted[c / kGroup] * kGroup + c % kGroup;
      w[q] = R::chunk(x, mis, a.cols, ch);
      i0[q] = ch * E - mis;
      float v[E];
      R::unpack(w[q], v);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i0[q] + e >= 0 && i0[q] + e < a.cols) best = max(best, order_key(v[e]) >> kShift);
    }
  }
  tau = bound(best);
  ties = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    if (__ballot(i0[q] < a.cols) == 0) continue;
    u32 key[E], mine = 0;
    float v[E];
    R::unpack(w[q], v);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool in = i0[q] + e >= 0 && i0[q] + e < a.cols;
      key[e] = in ? order_key(v[e]) >> kShift : 0;
      if (in && key[e] > tau) list[atomicAdd(&s_n[1], 1u)] = make_uint2(key[e], (u32)(i0[q] + e));
      mine += in && key[e] == tau;
    }
    u32 incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const u32 t = __shfl_up(incl, o);
      if (lane >= o) incl += t;
    }
    u32 at = ties + incl - mine;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool in = i0[q] + e >= 0 && i0[q] + e < a.cols;
      if (in && key[e] == tau && at++ < (u32)k) list[atomicAdd(&s_n[1], 1u)] = make_uint2(key[e], (u32)(i0[q] + e));
    }
    ties += __shfl(incl, 63);
  }
  __syncthreads();
  ranked(list, (int)s_n[1], k, [&](int r, uint2 c) {
    top_logp[r] = R::one(x + (int64_t)c.y * R::kEs) - m - log_s;
    top_ids[r] = c.y;
  });
}

static int seg_of(int64_t cols, int es) {
  const int e = 16 / es;
  // the row may start anywhere within its first chunk
  return (int)cdiv(cols + 2 * (e - 1), (int64_t)e * kThreads * kChunks);
}

template <Dt DT> static void launch(const Args& a, hipStream_t s) {
  hipLaunchKernelGGL((logprobs_segment_kernel<DT>), dim3((unsigned)(a.n_rows * a.n_seg)), dim3(kThreads), 0, s, a);
  // group maxima a lane of the second launch, or chunks' elements
  const int per = std::max(a.n_seg * (kThreads / kGroup * kChunks) / kThreads + 1,
                           kMaxTop * kGroup / kThreads * Row<DT>::kE);
  const size_t lds = a.top ? (size_t)list_cap(a.top, per) * sizeof(uint2) : 0;
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
  if (n_rows * a.n_seg > INT_MAX) return AAC_ERR_UNSUPPORTED;
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
