// Rotary positions (gfx950): the rotation of query and key heads by their tokens'
// angles, alone or on the way into the paged KV cache, and the cos / sin tables.
//
// A head's first R dims are R / 2 pairs, (d, d + R/2) or, interleaved, (2 d, 2 d + 1);
// pair d of a token at position p turns by the angle of row p, column d of the tables:
//   (x1, x2) -> (x1 c - x2 s, x1 s + x2 c), in fp32, rounded once to the head's type;
// dims from R on pass unchanged.  With caches, the rotated key and the value of new
// token i of sequence b go to the row that b's block table has for position
// cache_seqlens[b] + i (the k= / v= half of flash_attn_with_kvcache,
// model/model.py:233-240, for any number of new tokens).
//
// Bound by memory: every row is read and written once.  A wave takes one token's rows
// (query, key and value heads): CPR lanes a row, each with 8 pairs (two 16-byte vectors
// of 16-bit values), so the angles are loaded once for all the rows a lane takes and a
// pass over 64 / CPR rows needs no exchange between lanes.  PASSES passes go out before
// the first is used.
// 130 prompts of 17 to 4000 tokens (16/8 heads, bf16: 4.52 GB counted) 776 us, 5.8 TB/s;
// 16 x 4096 tokens of 32 heads (fp16, interleaved, 1.09 GB) 177 us, 6.2 TB/s, about what a
// copy of their size reaches (4.9 to 6.9); 256 tokens 4.6 us, latencies.

#include <algorithm>

#include "aac_common.h"

namespace aac {
namespace rot {

constexpr int kWaves = 4;
constexpr int64_t kMaxGroups = 1 << 24;  // of 256 threads: a launch numbers its threads in 32 bits

struct Rows {  // heads of one kind: element strides of a sequence, a token, a head
  const char* in;
  char* out;  // q: the rotated rows; k, v: the cache
  int64_t seq, tok, head;
  int64_t out_seq, out_tok, out_head;
  int32_t heads;
  int32_t len;  // tokens of a sequence that have such heads (without cu_seqlens)
};

struct Args {
  Rows q, k, v;
  const void* cos;
  const void* sin;
  int32_t table_rows, half;  // tables [table_rows, half]
  const int32_t* offsets;    // first position of a sequence, or null: offset0
  int32_t offset0;
  int32_t q_step;            // 0: every query of a sequence stands at its first position
  const int32_t* cu;         // packed tokens: their sequences' bounds, or null
  int32_t n_seqs;
  int32_t seqlen;            // tokens of a sequence (without cu)
  int64_t n_tokens;
  const int32_t* block_tables;
  int32_t max_blocks, block_size;
  int64_t num_blocks;
  int32_t dim;
  int32_t slots;  // waves a token
  int32_t sign;   // -1: turned back
  int32_t* context_lens;  // out, or null: first position + new keys
};

// Elements in their own type <-> fp32, N of them side by side.
template <Dt DT> struct Io;
template <> struct Io<Dt::FP32> {
  typedef float T;
  __device__ static inline float get(T x) { return x; }
  __device__ static inline T put(float x) { return x; }
};
template <> struct Io<Dt::BF16> {
  typedef u16 T;
  __device__ static inline float get(T x) { return __uint_as_float((u32)x << 16); }
  __device__ static inline T put(float x) { return (u16)Elem<Dt::BF16>::pack2_hw(x, x); }
};
template <> struct Io<Dt::FP16> {
  typedef u16 T;
  __device__ static inline float get(T x) { return (float)__builtin_bit_cast(_Float16, x); }
  __device__ static inline T put(float x) { return __builtin_bit_cast(u16, (_Float16)x); }
};

// 16 bytes; NT: non-temporal, past the caches.
template <bool NT> __device__ __forceinline__ u32x4 get16(const void* p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  else return *reinterpret_cast<const u32x4*>(p);
}
template <bool NT> __device__ __forceinline__ void put16(void* p, const u32x4& w) {
  if constexpr (NT) __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(p));
  else *reinterpret_cast<u32x4*>(p) = w;
}

// 16 bytes of elements <-> fp32: kN of them.
template <Dt DT> struct Vec {
  static constexpr int kN = 16 / Elem<DT>::kBytes;
  __device__ static inline void get(const u32x4& w, float* f) {
    if constexpr (DT == Dt::FP32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
    } else {
      Elem<DT>::unpack8(w, f);
    }
  }
  __device__ static inline u32x4 put(const float* f) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == Dt::FP32) w[i] = __float_as_uint(f[i]);
      else w[i] = Elem<DT>::pack2_hw(f[2 * i], f[2 * i + 1]);
    }
    return w;
  }
};

// K table values side by side, 8-byte aligned at least.
template <Dt DT, int K> __device__ __forceinline__ void table_values(const void* t, int64_t at, float* f) {
  typedef typename Io<DT>::T E;
  const E* p = reinterpret_cast<const E*>(t) + at;
  if constexpr (K * sizeof(E) % 16 == 0) {
#pragma unroll
    for (int i = 0; i < (int)(K * sizeof(E) / 16); ++i)
      Vec<DT>::get(reinterpret_cast<const u32x4*>(p)[i], f + i * Vec<DT>::kN);
  } else {
    static_assert(K * sizeof(E) == 8, "half a vector");
    const u32x2 w = *reinterpret_cast<const u32x2*>(p);
    float g[Vec<DT>::kN];
    Vec<DT>::get(u32x4{w[0], w[1], 0, 0}, g);
#pragma unroll
    for (int i = 0; i < K; ++i) f[i] = g[i];
  }
}

// The sequence of packed token t: the last b with cu[b] <= t (64 bounds a load).
__device__ __forceinline__ int seq_of(const int32_t* cu, int n_seqs, int64_t t, int lane) {
  int lo = 0, n = n_seqs;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int at = lane * step;
    const bool in = at < n && cu[lo + min(at, n - 1)] <= t;
    const int hits = __popcll(__ballot(in));
    const int skip = max(hits - 1, 0) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  return lo;
}

struct Place {
  int64_t q_at, in_at[3];  // element offsets of the token's rows: q out, q / k / v in
  int64_t crow;            // cache row of k and v, or -1
  int64_t s;               // number in its sequence
  int seq;
  int q_pos, k_pos;        // rows of the tables
  bool has_q, has_kv;
};

// Where a token's rows come from: known before its sequence and position are, so that
// they are on their way while those are looked up.
__device__ __forceinline__ void source_of(const Args& a, int64_t t, Place& p) {
  if (a.cu) {
    p.in_at[0] = t * a.q.tok;
    p.in_at[1] = t * a.k.tok;
    p.in_at[2] = t * a.v.tok;
    p.has_q = p.has_kv = true;
  } else {
    p.seq = (int)(t / a.seqlen);
    p.s = t - (int64_t)p.seq * a.seqlen;
    p.in_at[0] = p.seq * a.q.seq + p.s * a.q.tok;
    p.in_at[1] = p.seq * a.k.seq + p.s * a.k.tok;
    p.in_at[2] = p.seq * a.v.seq + p.s * a.v.tok;
    p.has_q = p.s < a.q.len;
    p.has_kv = p.s < a.k.len;
  }
}

// The token's position and where its rows go; false for a row of no sequence.
__device__ __forceinline__ bool target_of(const Args& a, int64_t t, int lane, Place& p) {
  if (a.cu) {
    p.seq = seq_of(a.cu, a.n_seqs, t, lane);
    p.s = t - a.cu[p.seq];
    if (p.s < 0 || t >= a.cu[p.seq + 1]) return false;
    p.q_at = t * a.q.out_tok;
  } else {
    p.q_at = p.seq * a.q.out_seq + p.s * a.q.out_tok;
  }
  const int64_t first = a.offsets ? a.offsets[p.seq] : a.offset0;
  if (a.context_lens && p.s == 0 && lane == 0) a.context_lens[p.seq] = (int)min(first + a.k.len, (int64_t)INT32_MAX);
  const int64_t last = max(a.table_rows - 1, 0);
  p.k_pos = (int)min(max(first + p.s, (int64_t)0), last);
  p.q_pos = (int)min(max(first + p.s * a.q_step, (int64_t)0), last);
  p.crow = -1;
  if (a.block_tables && p.has_kv) {
    const int64_t at = first + p.s;
    if (first >= 0 && at <= INT32_MAX && at < (int64_t)a.max_blocks * a.block_size) {
      const int blk = a.block_tables[(int64_t)p.seq * a.max_blocks + (int)at / a.block_size];
      if (blk >= 0 && blk < a.num_blocks) p.crow = (int64_t)blk * a.block_size + (int)at % a.block_size;
    }
  }
  return true;
}

// Row r of a token's heads (query, key, value heads in this order): its kind, its address
// in its tensor; -1 for a row the token lacks.
__device__ __forceinline__ int64_t row_in(const Args& a, const Place& p, int r, int& kind) {
  if (r < a.q.heads) {
    kind = 0;
    return p.has_q ? p.in_at[0] + r * a.q.head : -1;
  }
  r -= a.q.heads;
  kind = r < a.k.heads ? 1 : 2;
  r -= kind == 1 ? 0 : a.k.heads;
  return p.has_kv ? p.in_at[kind] + r * (kind == 1 ? a.k.head : a.v.head) : -1;
}
// where it goes; -1: nowhere
__device__ __forceinline__ int64_t row_out(const Args& a, const Place& p, int r, int kind) {
  if (kind == 0) return p.q_at + r * a.q.out_head;
  r -= a.q.heads + (kind == 1 ? 0 : a.k.heads);
  return p.crow >= 0 ? (p.crow * a.k.heads + r) * a.dim : -1;
}

// Two vectors of N elements a lane, placed so that a row's lanes read and write side by
// side: the two halves of N pairs, or N / 2 adjacent pairs each, or dims past them.  Head
// sizes of 2 N times a power of two up to 64, whole vectors of rotated dims, everything
// 16-byte aligned.
template <Dt DT, bool T32, bool INTER, int PASSES, bool NT>
__global__ __launch_bounds__(64 * kWaves) void rotary_kernel(Args a) {
  constexpr int ES = Elem<DT>::kBytes, N = Vec<DT>::kN;
  constexpr Dt TT = T32 ? Dt::FP32 : DT;
  const int lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = w / a.slots;
  if (t >= a.n_tokens) return;
  Place p;
  source_of(a, t, p);
  const int cpr = a.dim / (2 * N), c = lane & (cpr - 1), per = 64 / cpr;
  const int total = a.q.heads + a.k.heads + a.v.heads;
  // the lane's vectors in a row, and which of them are pairs
  const int rot = a.half / N;  // lanes whose vectors are halves of pairs (not INTER)
  int d0, d1;
  bool turn0, turn1;
  if (INTER) {
    d0 = N * c;
    d1 = d0 + a.dim / 2;
    turn0 = d0 < 2 * a.half;
    turn1 = d1 < 2 * a.half;
  } else {
    turn0 = turn1 = c < rot;
    d0 = N * c + (turn0 ? 0 : a.half);
    d1 = d0 + (turn0 ? a.half : N * (cpr - rot));
  }
  const int r0 = (int)(w - t * a.slots) * (PASSES * per) + lane / cpr;

  u32x4 x[PASSES][2];
  int kind[PASSES];
  bool live[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = r0 + i * per;
    const int64_t in = row_in(a, p, min(r, total - 1), kind[i]);
    live[i] = r < total && in >= 0;
    if (live[i]) {
      const char* src = (kind[i] == 0 ? a.q.in : kind[i] == 1 ? a.k.in : a.v.in) + in * ES;
      x[i][0] = get16<NT>(src + d0 * ES);
      x[i][1] = get16<NT>(src + d1 * ES);
    }
  }
  if (!target_of(a, t, lane, p)) return;
  // queries' and keys' angles: one row of the tables unless the queries all stand at
  // their sequence's first position
  float cf[N], sf[N];
  auto angles = [&](int pos) {
    const int64_t at = (int64_t)pos * a.half;
    if constexpr (INTER) {
      if (turn0) {
        table_values<TT, N / 2>(a.cos, at + d0 / 2, cf);
        table_values<TT, N / 2>(a.sin, at + d0 / 2, sf);
      }
      if (turn1) {
        table_values<TT, N / 2>(a.cos, at + d1 / 2, cf + N / 2);
        table_values<TT, N / 2>(a.sin, at + d1 / 2, sf + N / 2);
      }
    } else if (turn0) {
      table_values<TT, N>(a.cos, at + d0, cf);
      table_values<TT, N>(a.sin, at + d0, sf);
    }
    if (a.sign < 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) sf[i] = -sf[i];
    }
  };
  auto rotate = [](float& u, float& v, float cs, float sn) {
    const float u0 = u;
    u = fmaf(u0, cs, -(v * sn));
    v = fmaf(u0, sn, v * cs);
  };
  int have = -1;
  if (a.half > 0) angles(have = p.k_pos);
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int64_t out = row_out(a, p, r0 + i * per, kind[i]);
    if (!live[i] || out < 0) continue;
    if (kind[i] != 2 && a.half > 0) {
      const int pos = kind[i] == 0 ? p.q_pos : p.k_pos;
      if (pos != have) angles(have = pos);
      float f[N], g[N];
      Vec<DT>::get(x[i][0], f);
      Vec<DT>::get(x[i][1], g);
      if constexpr (INTER) {
        if (turn0) {
#pragma unroll
          for (int e = 0; e < N / 2; ++e) rotate(f[2 * e], f[2 * e + 1], cf[e], sf[e]);
          x[i][0] = Vec<DT>::put(f);
        }
        if (turn1) {
#pragma unroll
          for (int e = 0; e < N / 2; ++e) rotate(g[2 * e], g[2 * e + 1], cf[N / 2 + e], sf[N / 2 + e]);
          x[i][1] = Vec<DT>::put(g);
        }
      } else if (turn0) {
#pragma unroll
        for (int e = 0; e < N; ++e) rotate(f[e], g[e], cf[e], sf[e]);
        x[i][0] = Vec<DT>::put(f);
        x[i][1] = Vec<DT>::put(g);
      }
    }
    char* dst = (kind[i] == 0 ? a.q.out : kind[i] == 1 ? a.k.out : a.v.out) + out * ES;
    put16<NT>(dst + d0 * ES, x[i][0]);
    put16<NT>(dst + d1 * ES, x[i][1]);
  }
}

// The same for any even head size, rotated dims and alignment, an element pair a lane.
template <Dt DT, bool T32, bool INTER>
__global__ __launch_bounds__(64 * kWaves) void rotary_any_kernel(Args a) {
  typedef typename Io<DT>::T E;
  constexpr Dt TT = T32 ? Dt::FP32 : DT;
  typedef typename Io<TT>::T TE;
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= a.n_tokens) return;
  Place p;
  source_of(a, t, p);
  if (!target_of(a, t, lane, p)) return;
  const int total = a.q.heads + a.k.heads + a.v.heads, pairs = a.dim / 2;
  for (int64_t i = lane; i < (int64_t)total * pairs; i += 64) {
    const int r = (int)(i / pairs), c = (int)(i - (int64_t)r * pairs);
    int kind;
    const int64_t in = row_in(a, p, r, kind), out = row_out(a, p, r, kind);
    if (in < 0 || out < 0) continue;
    const bool pair = c < a.half;
    const int d0 = INTER || !pair ? 2 * c : c, d1 = INTER || !pair ? 2 * c + 1 : c + a.half;
    const E* src = reinterpret_cast<const E*>(kind == 0 ? a.q.in : kind == 1 ? a.k.in : a.v.in) + in;
    E* dst = reinterpret_cast<E*>(kind == 0 ? a.q.out : kind == 1 ? a.k.out : a.v.out) + out;
    E x0 = src[d0], x1 = src[d1];
    if (pair && kind != 2) {
      const int64_t at = (int64_t)(kind == 0 ? p.q_pos : p.k_pos) * a.half + c;
      const float cf = Io<TT>::get(reinterpret_cast<const TE*>(a.cos)[at]);
      const float sf = Io<TT>::get(reinterpret_cast<const TE*>(a.sin)[at]) * (float)a.sign;
      const float a0 = Io<DT>::get(x0), a1 = Io<DT>::get(x1);
      x0 = Io<DT>::put(fmaf(a0, cf, -(a1 * sf)));
      x1 = Io<DT>::put(fmaf(a0, sf, a1 * cf));
    }
    dst[d0] = x0;
    dst[d1] = x1;
  }
}

template <Dt DT, bool T32, bool INTER>
static int launch_i(Args a, bool fast, int n_cu, hipStream_t st) {
  if (!fast) {
    hipLaunchKernelGGL((rotary_any_kernel<DT, T32, INTER>), dim3((unsigned)cdiv(a.n_tokens, kWaves)),
                       dim3(64 * kWaves), 0, st, a);
    return AAC_OK;
  }
  const int per = 64 / (a.dim / (2 * Vec<DT>::kN)), total = a.q.heads + a.k.heads + a.v.heads;
  auto blocks_at = [&](int passes) {
    a.slots = (int)cdiv(total, (int64_t)per * passes);
    return cdiv(a.n_tokens * a.slots, kWaves);
  };
  // Many tokens: two passes a wave (260k tokens at 16/8 heads appended, us, 1 / 2 / 4 / 8
  // passes: 852 / 765 / 822 / 798).  What passes the caches anyway goes round them: 765
  // against 823, 16 x 4096 x 32 heads rotated 180 against 198.
  const bool many = total > per && a.n_tokens * cdiv(total, 2 * (int64_t)per) >= 8 * (int64_t)n_cu;
  const bool large = many && a.n_tokens * total * a.dim * Elem<DT>::kBytes >= (int64_t(64) << 20);
  const dim3 grid((unsigned)blocks_at(many ? 2 : 1)), block(64 * kWaves);
  if (large) hipLaunchKernelGGL((rotary_kernel<DT, T32, INTER, 2, true>), grid, block, 0, st, a);
  else if (many) hipLaunchKernelGGL((rotary_kernel<DT, T32, INTER, 2, false>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((rotary_kernel<DT, T32, INTER, 1, false>), grid, block, 0, st, a);
  return AAC_OK;
}

template <Dt DT>
static int launch_t(const Args& a, bool t32, bool inter, bool fast, int n_cu, hipStream_t st) {
  if constexpr (DT != Dt::FP32) {
    if (!t32)
      return inter ? launch_i<DT, false, true>(a, fast, n_cu, st) : launch_i<DT, false, false>(a, fast, n_cu, st);
  }
  return inter ? launch_i<DT, true, true>(a, fast, n_cu, st) : launch_i<DT, true, false>(a, fast, n_cu, st);
}

static int launch(const Args& a, int32_t table_dtype, bool inter, int32_t dtype, hipStream_t st) {
  const int es = dtype == AAC_DTYPE_FP32 ? 4 : 2, ts = table_dtype == AAC_DTYPE_FP32 ? 4 : 2;
  const int n = 16 / es, cpr = a.dim / (2 * n), unit = inter ? n / 2 : n;
  // every vector the fast kernel touches: rows, heads and tables at multiples of 16 bytes
  // (interleaved pairs: tables of half vectors)
  bool fast = a.dim % (2 * n) == 0 && (cpr & (cpr - 1)) == 0 && cpr <= 64 && a.half % unit == 0 &&
              (((uintptr_t)a.cos | (uintptr_t)a.sin) % 16) == 0 && a.half * ts % std::min(16, unit * ts) == 0;
  for (const Rows* r : {&a.q, &a.k, &a.v})
    if (r->heads) {
      fast = fast && (((uintptr_t)r->in | (uintptr_t)r->out) % 16) == 0;
      for (int64_t s : {r->seq, r->tok, r->head, r->out_seq, r->out_tok, r->out_head}) fast = fast && s * es % 16 == 0;
    }
  // Waves of so many tokens: the fast kernel's take two passes where one does not do.
  if (a.n_tokens > kWaves * (kMaxGroups - 1)) return AAC_ERR_UNSUPPORTED;
  const int64_t heads = (int64_t)a.q.heads + a.k.heads + a.v.heads, per = fast ? 64 / cpr : heads;
  if (cdiv(a.n_tokens * (heads > per ? cdiv(heads, 2 * per) : 1), kWaves) >= kMaxGroups) return AAC_ERR_UNSUPPORTED;
  int n_cu = 0;
  int rc = device_cu_count(&n_cu);
  if (rc != AAC_OK) return rc;
  const bool t32 = table_dtype == AAC_DTYPE_FP32;
  switch (dtype) {
    case AAC_DTYPE_BF16: rc = launch_t<Dt::BF16>(a, t32, inter, fast, n_cu, st); break;
    case AAC_DTYPE_FP16: rc = launch_t<Dt::FP16>(a, t32, inter, fast, n_cu, st); break;
    default: rc = launch_t<Dt::FP32>(a, t32, inter, fast, n_cu, st); break;
  }
  if (rc != AAC_OK) return rc;
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? AAC_OK : (int)e;
}

// Arguments both entry points check alike.
static int check_tables(const void* cos, const void* sin, int32_t rows, int32_t rotary_dim, int32_t table_dtype,
                        int32_t head_dim, int32_t dtype) {
  if (dtype != AAC_DTYPE_BF16 && dtype != AAC_DTYPE_FP16 && dtype != AAC_DTYPE_FP32) return AAC_ERR_UNSUPPORTED;
  if (head_dim <= 0 || rotary_dim < 0 || rows < 0) return AAC_ERR_INVALID_ARGUMENT;
  if (head_dim % 2 || rotary_dim % 2 || rotary_dim > head_dim) return AAC_ERR_SHAPE;
  if (rotary_dim == 0) return AAC_OK;
  if (table_dtype != AAC_DTYPE_FP32 && table_dtype != dtype) return AAC_ERR_UNSUPPORTED;
  if (!cos || !sin || rows == 0) return AAC_ERR_INVALID_ARGUMENT;
  return AAC_OK;
}

// ------------------------------------------------------------------ tables
// cos and sin of position p, frequency i: the angle in quarter turns, 4 p turns[i], less the
// nearest whole number of them, in fp64 (at position 2^20 a radian keeps 2^-33 of
// precision there, 2^-4 in fp32); what remains is within an eighth of a turn, and its
// sine and cosine are polynomials in fp32, near-minimax from interpolation at Chebyshev
// nodes (truncation below 1e-10, with their rounding 8.5e-8 at most; root mean square 4.1e-8 of
// the values where the same in fp64, rounded once, has 2.9e-8).  The whole number's last
// bits, the quadrant, are the low bits of its sum with 1.5 * 2^52.
// A vector of each a thread: 131,072 x 64 in fp32 11.3-13.4 us (67 MB, 5 TB/s and more).
__device__ __forceinline__ void cos_sin_of(double x, float factor, float& c, float& s) {
  constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52
  const double y = x + kRound;
  const float r = (float)(x - (y - kRound)), u = r * r;
  const u32 quad = (u32)(uint64_t)__double_as_longlong(y);
  const float sn = r * factor * fmaf(u, fmaf(u, fmaf(u, fmaf(u, 0.00015820628f, -0.0046812664f), 0.07969258f), -0.6459641f), 1.5707964f);
  const float cn = factor * fmaf(u, fmaf(u, fmaf(u, fmaf(u, 0.00090362807f, -0.02086007f), 0.2536692f), -1.2337005f), 1.0f);
  const float a = quad & 1 ? sn : cn, b = quad & 1 ? cn : sn;
  c = __uint_as_float(__float_as_uint(a) ^ ((quad + 1) << 30 & 0x80000000u));
  s = __uint_as_float(__float_as_uint(b) ^ (quad << 30 & 0x80000000u));
}

template <Dt DT>
__global__ __launch_bounds__(256) void tables_kernel(const double* turns, int32_t half, const int32_t* positions,
                                                     int64_t start, int64_t n, float factor, void* cos_out,
                                                     void* sin_out) {
  typedef typename Io<DT>::T E;
  constexpr int N = Vec<DT>::kN;
  const u32 groups = (half + N - 1) / N;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n * groups) return;
  const int64_t r = i >> 32 ? i / groups : (int64_t)((u32)i / groups);
  const int f0 = (int)(i - r * groups) * N;
  const double pos = 4.0 * (double)(positions ? (int64_t)positions[r] : start + r);
  float c[N], s[N];
#pragma unroll
  for (int e = 0; e < N; ++e) cos_sin_of(pos * turns[min(f0 + e, half - 1)], factor, c[e], s[e]);
  E* co = reinterpret_cast<E*>(cos_out) + r * half + f0;
  E* so = reinterpret_cast<E*>(sin_out) + r * half + f0;
  if (half % N == 0) {
    *reinterpret_cast<u32x4*>(co) = Vec<DT>::put(c);
    *reinterpret_cast<u32x4*>(so) = Vec<DT>::put(s);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (f0 + e < half) {
        co[e] = Io<DT>::put(c[e]);
        so[e] = Io<DT>::put(s[e]);
      }
  }
}

}  // namespace rot
}  // namespace aac

using namespace aac;

extern "C" int aac_rotary(const void* x, int64_t x_seq_stride, int64_t x_tok_stride, int64_t x_head_stride,
                          void* out, int64_t out_seq_stride, int64_t out_tok_stride, int64_t out_head_stride,
                          int32_t n_seqs, int32_t seqlen, int64_t n_tokens, const int32_t* cu_seqlens,
                          const int32_t* offsets, int32_t offset, int32_t n_heads, int32_t head_dim,
                          const void* cos_table, const void* sin_table, int32_t table_rows, int32_t rotary_dim,
                          int32_t interleaved, int32_t conjugate, int32_t table_dtype, int32_t dtype,
                          void* stream) {
  int rc = rot::check_tables(cos_table, sin_table, table_rows, rotary_dim, table_dtype, head_dim, dtype);
  if (rc != AAC_OK) return rc;
  if (n_seqs < 0 || seqlen < 0 || n_tokens < 0 || n_heads < 0) return AAC_ERR_INVALID_ARGUMENT;
  if (!cu_seqlens) n_tokens = (int64_t)n_seqs * seqlen;
  if (n_tokens == 0 || n_seqs == 0 || n_heads == 0) return AAC_OK;
  if (!x || !out) return AAC_ERR_INVALID_ARGUMENT;
  rot::Args a = {};
  a.q = {(const char*)x, (char*)out, x_seq_stride, x_tok_stride, x_head_stride, out_seq_stride, out_tok_stride,
         out_head_stride, n_heads, seqlen};
  a.cos = cos_table;
  a.sin = sin_table;
  a.table_rows = table_rows;
  a.half = rotary_dim / 2;
  a.offsets = offsets;
  a.offset0 = offset;
  a.q_step = 1;
  a.cu = cu_seqlens;
  a.n_seqs = n_seqs;
  a.seqlen = std::max(seqlen, 1);
  a.n_tokens = n_tokens;
  a.dim = head_dim;
  a.sign = conjugate ? -1 : 1;
  return rot::launch(a, rotary_dim ? table_dtype : (int32_t)AAC_DTYPE_FP32, interleaved != 0, dtype,
                     (hipStream_t)stream);
}

extern "C" int aac_rotary_append_paged(
    const void* q, int64_t q_seq_stride, int64_t q_tok_stride, int64_t q_head_stride, const void* k,
    int64_t k_seq_stride, int64_t k_tok_stride, int64_t k_head_stride, const void* v, int64_t v_seq_stride,
    int64_t v_tok_stride, int64_t v_head_stride, void* q_out, int32_t n_seqs, int32_t seqlen_q, int32_t seqlen_k,
    int64_t n_tokens, const int32_t* cu_seqlens, const int32_t* cache_seqlens, int32_t* context_lens, int32_t n_q_heads,
    int32_t n_kv_heads, int32_t head_dim, const void* cos_table, const void* sin_table, int32_t table_rows,
    int32_t rotary_dim, int32_t interleaved, int32_t queries_at_first, void* k_cache, void* v_cache,
    int64_t num_blocks, int32_t block_size, const int32_t* block_tables, int32_t max_blocks_per_seq,
    int32_t table_dtype, int32_t dtype, void* stream) {
  int rc = rot::check_tables(cos_table, sin_table, table_rows, rotary_dim, table_dtype, head_dim, dtype);
  if (rc != AAC_OK) return rc;
  if (n_seqs < 0 || seqlen_q < 0 || seqlen_k < 0 || n_tokens < 0 || n_q_heads < 0 || n_kv_heads <= 0 ||
      num_blocks < 0 || block_size <= 0 || max_blocks_per_seq <= 0)
    return AAC_ERR_INVALID_ARGUMENT;
  const int32_t seqlen = std::max(q ? seqlen_q : 0, seqlen_k);
  if (!cu_seqlens) n_tokens = (int64_t)n_seqs * seqlen;
  if (n_tokens == 0 || n_seqs == 0) return AAC_OK;
  if (!k || !v || !k_cache || !v_cache || !block_tables || !cache_seqlens || (q && !q_out))
    return AAC_ERR_INVALID_ARGUMENT;
  rot::Args a = {};
  if (q && n_q_heads)
    a.q = {(const char*)q, (char*)q_out, q_seq_stride, q_tok_stride, q_head_stride,
           (int64_t)seqlen_q * n_q_heads * head_dim, (int64_t)n_q_heads * head_dim, head_dim, n_q_heads, seqlen_q};
  a.k = {(const char*)k, (char*)k_cache, k_seq_stride, k_tok_stride, k_head_stride, 0, 0, head_dim, n_kv_heads,
         seqlen_k};
  a.v = {(const char*)v, (char*)v_cache, v_seq_stride, v_tok_stride, v_head_stride, 0, 0, head_dim, n_kv_heads,
         seqlen_k};
  a.cos = cos_table;
  a.sin = sin_table;
  a.table_rows = table_rows;
  a.half = rotary_dim / 2;
  a.offsets = cache_seqlens;
  a.q_step = queries_at_first ? 0 : 1;
  a.cu = cu_seqlens;
  a.n_seqs = n_seqs;
  a.seqlen = std::max(seqlen, 1);
  a.n_tokens = n_tokens;
  a.context_lens = cu_seqlens ? nullptr : context_lens;
  a.block_tables = block_tables;
  a.max_blocks = max_blocks_per_seq;
  a.block_size = block_size;
  a.num_blocks = num_blocks;
  a.dim = head_dim;
  a.sign = 1;
  return rot::launch(a, rotary_dim ? table_dtype : (int32_t)AAC_DTYPE_FP32, interleaved != 0, dtype,
                     (hipStream_t)stream);
}

extern "C" int aac_rotary_tables(const void* turns, int32_t n_freqs, const int32_t* positions, int64_t start,
                                 int64_t n_positions, float factor, void* cos_out, void* sin_out, int32_t dtype,
                                 void* stream) {
  if (dtype != AAC_DTYPE_BF16 && dtype != AAC_DTYPE_FP16 && dtype != AAC_DTYPE_FP32) return AAC_ERR_UNSUPPORTED;
  if (n_freqs <= 0 || n_positions < 0) return AAC_ERR_INVALID_ARGUMENT;
  if (n_positions == 0) return AAC_OK;
  if (!turns || !cos_out || !sin_out) return AAC_ERR_INVALID_ARGUMENT;
  const int vec = dtype == AAC_DTYPE_FP32 ? 4 : 8;
  if (n_freqs % vec == 0 && ((uintptr_t)cos_out | (uintptr_t)sin_out) % 16) return AAC_ERR_MISALIGNED;
  // (positions are whole numbers in fp64, and their product with 4 turns has a quadrant)
  if (start < -(int64_t(1) << 40) || start > (int64_t(1) << 40)) return AAC_ERR_SHAPE;
  const int64_t blocks = cdiv(n_positions * cdiv(n_freqs, vec), 256);
  if (n_positions >= (int64_t(1) << 40) / n_freqs || blocks >= rot::kMaxGroups) return AAC_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)blocks), block(256);
  const double* f = (const double*)turns;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case AAC_DTYPE_BF16:
      hipLaunchKernelGGL((rot::tables_kernel<Dt::BF16>), grid, block, 0, st, f, n_freqs, positions, start, n_positions,
                         factor, cos_out, sin_out);
      break;
    case AAC_DTYPE_FP16:
      hipLaunchKernelGGL((rot::tables_kernel<Dt::FP16>), grid, block, 0, st, f, n_freqs, positions, start, n_positions,
                         factor, cos_out, sin_out);
      break;
    default:
      hipLaunchKernelGGL((rot::tables_kernel<Dt::FP32>), grid, block, 0, st, f, n_freqs, positions, start, n_positions,
                         factor, cos_out, sin_out);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? AAC_OK : (int)e;
}
