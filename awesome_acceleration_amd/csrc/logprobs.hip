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
// Two launches.  The first cuts a row into segments that a workgroup holds in its
// registers (16 KiB of packed values in 256 threads x 8 chunks of 16 bytes), so the
// logits are read once and gone over several times: the segment's maximum, the sums
// about it, then the candidates of the top k.  A bound for those: in a wave, the k-th
// largest of the 64 lanes' maxima (found bit by bit with ballots) has at least k values
// of the segment at or above it; the largest such bound of the four waves holds for
// the segment.  Values above it go to a list in LDS; of those equal to it each wave adds
// the first k in index order (a masked row is -inf nearly everywhere).  A list
// that a wave's share of would not hold (values sorted across the lanes) is replaced
// by k selections over the registers.  The second launch merges a row's segments.
// Bound by the read of the logits.
#include <algorithm>
#include <climits>

#include "aac_common.h"

namespace aac {
namespace lp {

constexpr int kThreads = 256;
constexpr int kChunks = 8;     // 16-byte chunks a thread
constexpr int kMaxTop = 32;
constexpr int kWaveCap = 192;  // candidates above the bound a wave may list

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
  float* ws_sum;   // [n_rows, n_seg, 4]: m, S, T
  uint2* ws_top;   // [n_rows, n_seg, top]: value bits, index
};

template <Dt DT> struct Row {
  static constexpr int kEs = DT == Dt::FP32 ? 4 : 2;
  static constexpr int kE = 16 / kEs;  // elements of a chunk
  static constexpr int kSegChunks = kThreads * kChunks;
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
};

// chunks of a row: the row starts `mis` elements into its first one
__host__ __device__ inline int64_t n_chunks(int64_t cols, int mis, int e) { return (cols + mis + e - 1) / e; }

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
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
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
  const int64_t nch = n_chunks(a.cols, mis, E);
  const int64_t c0 = (int64_t)seg * R::kSegChunks + tid;  // chunk c0 + 256 u
  // index of the first element of chunk u
  auto first = [&](int u) { return (c0 + kThreads * u) * E - mis; };

  u32x4 w[kChunks];
  constexpr u32 kNone = DT == Dt::BF16 ? 0xff80ff80u : DT == Dt::FP16 ? 0xfc00fc00u : 0xff800000u;
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    const int64_t i0 = first(u);
    if (i0 >= 0 && i0 + E <= a.cols) {
      w[u] = *reinterpret_cast<const u32x4*>(p + i0 * R::kEs);
    } else {  // past the row (-inf: adds nothing), or its first or last elements
      w[u] = u32x4{kNone, kNone, kNone, kNone};
      if (c0 + kThreads * u < nch) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int64_t i = i0 + e;
          if (i < 0 || i >= a.cols) continue;
          if constexpr (DT == Dt::FP32) {
            w[u][e] = *reinterpret_cast<const u32*>(p + i * 4);
          } else {
            const u32 b = *reinterpret_cast<const u16*>(p + i * 2);
            w[u][e >> 1] = e & 1 ? (w[u][e >> 1] & 0xffffu) | b << 16 : (w[u][e >> 1] & 0xffff0000u) | b;
          }
        }
      }
    }
  }

  // maxima of the chunks (NaN if one is), the thread, the segment
  float cm[kChunks], tm = -INFINITY;
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    float v[E];
    R::unpack(w[u], v);
    cm[u] = v[0];
#pragma unroll
    for (int e = 1; e < E; ++e) cm[u] = vmax(cm[u], v[e]);
    tm = vmax(tm, cm[u]);
  }
  __shared__ float sm[3][4];
  float m = tm;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = vmax(m, __shfl_xor(m, o));
  if (lane == 0) sm[0][wave] = m;

  // the wave's bound for the top k
  __shared__ u32 s_tau[4], s_cnt[4], s_over;
  u32 tau = 0;
  if (a.top > 0) {
    const u32 key = order_key(tm);
#pragma unroll 1
    for (u32 bit = 0x80000000u; bit; bit >>= 1) {
      const u32 t = tau | bit;
      if ((int)__popcll(__ballot(key >= t)) >= a.top) tau = t;
    }
    if (lane == 0) {
      s_tau[wave] = tau;
      s_cnt[wave] = 0;
    }
    if (tid == 0) s_over = 0;
  }
  __syncthreads();
  m = vmax(vmax(sm[0][0], sm[0][1]), vmax(sm[0][2], sm[0][3]));
  tau = max(max(s_tau[0], s_tau[1]), max(s_tau[2], s_tau[3]));

  // sums about the segment's maximum
  float S = 0.f, T = 0.f;
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    float v[E];
    R::unpack(w[u], v);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = fmaxf(v[e] - m, -1e30f);  // (-inf and -inf - -inf: adds 0)
      const float p = fast_exp2(d * kLog2e);
      S += p;
      T = fmaf(p, d, T);
    }
  }
  S = wave_sum(S);
  T = wave_sum(T);
  if (lane == 0) {
    sm[1][wave] = S;
    sm[2][wave] = T;
  }

  // candidates
  __shared__ uint2 list[4][kWaveCap + kMaxTop];
  if (a.top > 0) {
    u32 above = 0, ties = 0;  // uniform in the wave
#pragma unroll
    for (int u = 0; u < kChunks; ++u) {
      if (__ballot(order_key(cm[u]) >= tau) == 0) continue;
      float v[E];
      R::unpack(w[u], v);
      const int64_t i0 = first(u);
      u32 mine = 0;  // this lane's ties in the chunk
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const bool in = i0 + e >= 0 && i0 + e < a.cols;
        const u32 key = order_key(v[e]);
        const unsigned long long bal = __ballot(in && key > tau);
        if (in && key > tau) {
          const u32 at = above + __builtin_amdgcn_mbcnt_hi((u32)(bal >> 32), __builtin_amdgcn_mbcnt_lo((u32)bal, 0u));
          if (at < kWaveCap) list[wave][at] = make_uint2(__float_as_uint(v[e]), (u32)(i0 + e));
        }
        above += (u32)__popcll(bal);
        mine += in && key == tau;
      }
      if (ties < (u32)a.top) {
        u32 incl = mine;  // ties in index order: lane by lane
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const u32 t = __shfl_up(incl, o);
          if (lane >= o) incl += t;
        }
        u32 at = ties + incl - mine;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const bool in = i0 + e >= 0 && i0 + e < a.cols;
          if (in && order_key(v[e]) == tau) {
            if (at < (u32)a.top) list[wave][kWaveCap + at] = make_uint2(__float_as_uint(v[e]), (u32)(i0 + e));
            ++at;
          }
        }
        ties += __shfl(incl, 63);
      }
    }
    ties = min(ties, (u32)a.top);
    if (above > (u32)kWaveCap) {
      if (lane == 0) s_over = 1;
    } else {
      // ties behind the values above the bound, in one piece
      uint2 t = make_uint2(0, 0);
      if ((u32)lane < ties) t = list[wave][kWaveCap + lane];
      if ((u32)lane < ties) list[wave][above + lane] = t;
    }
    if (lane == 0) s_cnt[wave] = above + ties;
  }
  __syncthreads();
  if (tid == 0) {
    float* o = a.ws_sum + (row * a.n_seg + seg) * 4;
    o[0] = m;
    o[1] = sm[1][0] + sm[1][1] + sm[1][2] + sm[1][3];
    o[2] = sm[2][0] + sm[2][1] + sm[2][2] + sm[2][3];
  }
  if (a.top == 0) return;
  uint2* out = a.ws_top + (row * a.n_seg + seg) * a.top;
  if (!s_over) {  // each candidate's rank
    const int n0 = s_cnt[0], n1 = n0 + s_cnt[1], n2 = n1 + s_cnt[2], n = n2 + s_cnt[3];
    for (int i = tid; i < max(n, a.top); i += kThreads) {
      if (i >= n) {  // fewer values than k in the segment
        out[i] = make_uint2(0, 0xffffffffu);
        continue;
      }
      const int q = (i >= n0) + (i >= n1) + (i >= n2);
      const uint2 c = list[q][i - (q == 0 ? 0 : q == 1 ? n0 : q == 2 ? n1 : n2)];
      const u32 k = order_key(__uint_as_float(c.x));
      int rank = 0;
      for (int r = 0; r < 4; ++r)
        for (u32 z = 0; z < s_cnt[r]; ++z) {
          const uint2 d = list[r][z];
          rank += before(order_key(__uint_as_float(d.x)), d.y, k, c.y);
        }
      if (rank < a.top) out[rank] = c;
    }
    return;
  }
  // k selections: the best value behind the one selected last
  __shared__ uint2 s_best[4];
  u32 lk = 0xffffffffu, li = 0;
  bool any = false;
  for (int r = 0; r < a.top; ++r) {
    u32 bk = 0, bi = 0xffffffffu, bv = 0;
#pragma unroll
    for (int u = 0; u < kChunks; ++u) {
      float v[E];
      R::unpack(w[u], v);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int64_t i = first(u) + e;
        const u32 key = order_key(v[e]);
        if (i >= 0 && i < a.cols && (!any || before(lk, li, key, (u32)i)) && before(key, (u32)i, bk, bi)) {
          bk = key;
          bi = (u32)i;
          bv = __float_as_uint(v[e]);
        }
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const u32 ok = __shfl_xor(bk, o), oi = __shfl_xor(bi, o), ov = __shfl_xor(bv, o);
      if (before(ok, oi, bk, bi)) {
        bk = ok;
        bi = oi;
        bv = ov;
      }
    }
    if (lane == 0) s_best[wave] = make_uint2(bv, bi);
    __syncthreads();
    uint2 best = make_uint2(0, 0xffffffffu);
    u32 best_k = 0;
    for (int q = 0; q < 4; ++q) {
      const u32 k = s_best[q].y == 0xffffffffu ? 0 : order_key(__uint_as_float(s_best[q].x));
      if (before(k, s_best[q].y, best_k, best.y)) {
        best = s_best[q];
        best_k = k;
      }
    }
    if (tid == 0) out[r] = best;
    if (best.y != 0xffffffffu) {
      lk = best_k;
      li = best.y;
      any = true;
    }
    __syncthreads();
  }
}

// A row's segments: the sums, and the top k of the sorted lists (a candidate's rank is
// its place in its own list plus, by bisection, the better ones in each other list).
template <Dt DT>
__global__ __launch_bounds__(kThreads) void logprobs_merge_kernel(Args a) {
  typedef Row<DT> R;
  extern __shared__ uint2 cand[];  // [n_seg * top]
  __shared__ float s_log;
  __shared__ float s_m;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, n = a.n_seg * a.top;
  for (int i = tid; i < n; i += kThreads) cand[i] = a.ws_top[row * n + i];
  if (tid < 64) {
    const float* p = a.ws_sum + row * a.n_seg * 4;
    float m = -INFINITY;
    for (int s = tid; s < a.n_seg; s += 64) m = vmax(m, p[4 * s]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = vmax(m, __shfl_xor(m, o));
    float S = 0.f, T = 0.f;
    for (int s = tid; s < a.n_seg; s += 64) {
      const float d = fmaxf(p[4 * s] - m, -1e30f);
      const float f = fast_exp2(d * kLog2e);
      S = fmaf(p[4 * s + 1], f, S);
      T += f * fmaf(d, p[4 * s + 1], p[4 * s + 2]);
    }
    S = wave_sum(S);
    T = wave_sum(T);
    const bool none = !(fabsf(m) < INFINITY);
    const float log_s = none ? __uint_as_float(0x7fc00000u) : logf(S);
    if (tid == 0) {
      s_log = log_s;
      s_m = m;
      a.entropy[row] = log_s - T / S;
      const int64_t t = a.tokens[row];
      float lp = 0.f;  // a negative token is padding
      if (t >= a.cols) lp = __uint_as_float(0x7fc00000u);
      else if (t >= 0) lp = R::one(a.x + row * a.stride + t * R::kEs) - m - log_s;
      a.logp[row] = lp;
    }
  }
  __syncthreads();
  for (int i = tid; i < n; i += kThreads) {
    const uint2 c = cand[i];
    if (c.y == 0xffffffffu) continue;
    const u32 k = order_key(__uint_as_float(c.x));
    const int own = i / a.top;
    int rank = i - own * a.top;
    for (int s = 0; s < a.n_seg && rank < a.top; ++s) {
      if (s == own) continue;
      int lo = 0, hi = a.top;  // entries before lo are better, from hi on are not
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        const uint2 d = cand[s * a.top + mid];
        if (d.y != 0xffffffffu && before(order_key(__uint_as_float(d.x)), d.y, k, c.y)) lo = mid + 1;
        else hi = mid;
      }
      rank += lo;
    }
    if (rank < a.top) {
      a.top_logp[row * a.top + rank] = __uint_as_float(c.x) - s_m - s_log;
      a.top_ids[row * a.top + rank] = c.y;
    }
  }
}

static int seg_of(int64_t cols, int es) {
  const int e = 16 / es;
  // the row may start anywhere within its first chunk
  return (int)cdiv(n_chunks(cols, e - 1, e), kThreads * kChunks);
}

template <Dt DT> static void launch(const Args& a, hipStream_t s) {
  hipLaunchKernelGGL((logprobs_segment_kernel<DT>), dim3((unsigned)(a.n_rows * a.n_seg)), dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL((logprobs_merge_kernel<DT>), dim3((unsigned)a.n_rows), dim3(kThreads),
                     (size_t)a.n_seg * a.top * sizeof(uint2), s, a);
}

}  // namespace lp
}  // namespace aac

using namespace aac;

extern "C" size_t aac_logprobs_workspace_bytes(int64_t n_rows, int64_t n_cols, int32_t top_k) {
  if (n_rows <= 0 || n_cols <= 0 || top_k < 0) return 0;
  const size_t segs = (size_t)n_rows * lp::seg_of(n_cols, 4);  // fp32 rows have the most segments
  return segs * 16 + segs * top_k * sizeof(uint2);
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
  a.ws_top = (uint2*)((char*)workspace + (size_t)n_rows * a.n_seg * 16);
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case AAC_DTYPE_BF16: lp::launch<Dt::BF16>(a, s); break;
    case AAC_DTYPE_FP16: lp::launch<Dt::FP16>(a, s); break;
    default: lp::launch<Dt::FP32>(a, s); break;
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? AAC_OK : (int)e;
}
