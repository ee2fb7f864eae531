// Attention of a chunk of new tokens over the paged KV cache (gfx950, bf16/fp16 MFMA):
// sequence b's n_b queries see its L_b cached tokens (the new ones among them) through
// its block table, causal ones the first i + 1 + L_b - n_b of them.  The calls between a
// prefill (llm.py:178-184) and a decode step (model/model.py:233-240): chunked prefill,
// the next turn of a conversation, draft tokens to verify.
//
// A KV head's queries are rows: row r is query r / G of head r % G of its group, so any
// group size fills the matrix tiles and every key read serves all of them.  A wave holds
// 32 rows; S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16, the layouts, lazy
// rescaling and rounding of the probabilities as in prefill_split.hip.  A workgroup is R
// row blocks times SL key slices: the slices of a row block take 32-key sub-tiles s, s +
// SL, ... and are merged through LDS at the end.
//
// Pages.  16 keys of a tile lie in one page (block sizes are multiples of 16, or one
// block holds the sequence), so a wave finds their address with scalar loads and
// arithmetic, one iteration ahead, and brings them with direct loads into LDS through a
// buffer resource that ends at the context: rows behind it, whatever the page holds,
// arrive as zeros.  Other block sizes look every row up in its lane, right before its load
// (PAGE16 false); the wait for the entry is one for all loads in flight, so nothing overlaps
// there: pages of 20 / 40 tokens against 16, us, 777 queries over 7778 keys at 16/8 heads 86 /
// 86 against 69, 16 x 5 over 1.0-2.0k 39 / 39 against 27, 4 x 1024 over 8192 at 32/8 570 / 566
// against 463.
//
// Roundings.  Scores, softmax statistics and sums are fp32; the probabilities are rounded to
// 16 bits once, the second product's operands (a second term for what that loses would cost
// another of these products), and the row sum is of the rounded ones, so that the weights add
// up to 1.  The reciprocal is the hardware's, a unit of 2^-23 off.  Against 64 bits outputs
// are 2.0e-3 off in bf16 (root mean square, relative; fp32 throughout and rounded once at the
// end 1.7e-3), 2.6e-4 in fp16 (2.1e-4).
//
// Queries.  A wave's rows come in the same way, into the place of the ring's last stages,
// beside the first stages' keys (loaded to registers, with every load waited for at the
// start, calls of 97 to 306 tokens took 8.2-19 us where they take 7.6-17.5).  What depends on the lane alone is
// worked out again for each item of shared work: kept, 18 vector registers of the 256-row
// form spilled.  Two still do with pages that are no multiple of 16; the shared forms keep up
// to 35 scalar registers in vector lanes.
//
// Bounds.  8 sequences of 2048 over 14-30k keys at 32/8 heads (6.12 TFLOP) take 5.43-5.48
// ms, 1.12 PFLOP/s at the 1.9 GHz that the card holds there: 1.88 us for the 64 keys of
// an iteration and 256 rows.  The matrix units are busy 56% of it; two waves a SIMD overlap
// their products, LDS reads (32 KiB a wave) and softmax in part (copies without the softmax
// took 4.28 ms, without LDS reads 4.88, without loads 5.30; 915 MB are read from HBM, each
// key once).  Worse: the waves of a SIMD in turns by barriers 5.85, fragments refilled between
// the products 6.18, a sub-tile's products beside the other's softmax 6.1.  777 queries over 7778
// keys at 16/8 68-75 us, 10 of them the join; 16 x 5 over 1.0-2.0k 28, latencies.
//
// Few or uneven sequences: the workgroups share the work out evenly (below).

#include <algorithm>

#include "prefill_common.h"

namespace aac {
namespace pp {

using pf::D;
using pf::kRescale;

constexpr int kSubBytes = 32 * D * 2;  // 8 KiB: 32 keys of K or V
constexpr int kOutPitch = D * 2 + 16;

struct Args {
  const u16* q;
  const u16* kc;
  const u16* vc;
  u16* out;
  int64_t q_stride, o_stride;
  const int32_t* cu_q;
  const int32_t* ctx;   // context lengths, or null:
  const int32_t* cu_k;  // their prefix sums
  const int32_t* tables;
  int64_t n_tokens;
  u32 num_blocks;       // those an int32 table can name
  int32_t n_seqs, hq, hkv, group;
  u32 group31;          // ceil(2^31 / group)
  int32_t max_q;        // queries of every sequence where cu_q is null
  int32_t block_size, max_blocks;
  int32_t capacity;     // keys a table can name
  u32 magic, shift;     // 16-key group -> page (PAGE16), key -> page otherwise
  int32_t row_bytes;    // of a cache row, all heads
  float scale_log2;
  int32_t n_rb;         // row blocks of the longest sequence
  float* ws_o;          // shared work: [workgroup][2][row blocks][4][4][64 lanes][4]
  float2* ws_ml;        // [workgroup][2][row blocks][32]
  struct Cut* ws_cut;   // [workgroup]
};

// The item at the start of a share, for the kernel that joins its parts: those of shares
// first to last, where they are two or more and this is the item's first cut; share
// `opens` holds its beginning.
struct Cut {
  int first, last, opens, row0, rows, q_beg, pad[2];  // (32 bytes)
};

// x / d for x < 2^27: x * ceil(2^(27 + s) / d) >> (27 + s), s = ceil(log2 d).
__device__ __forceinline__ int divide(const Args& a, int x) { return (int)(((uint64_t)(u32)x * a.magic) >> a.shift); }

struct Seq {
  int q_beg, Lq, Lk;
  // rows of a KV head (of more queries than the call says, as many as an int holds)
  __device__ __forceinline__ int rows(const Args& a) const {
    return Lq > 0 ? (int)min((int64_t)Lq * a.group, (int64_t)1 << 30) : 0;
  }
};
__device__ __forceinline__ Seq seq_of(const Args& a, int s) {
  typedef const int32_t __attribute__((address_space(4))) cint;  // scalar loads
  const cint* cu = (const cint*)(uintptr_t)a.cu_q;
  Seq r;
  if (a.cu_q) {
    r.q_beg = max(cu[s], 0);
    r.Lq = (int)min((int64_t)cu[s + 1], a.n_tokens) - r.q_beg;
  } else {
    r.q_beg = s * a.max_q;
    r.Lq = a.max_q;
  }
  int lk;
  if (a.ctx) {
    lk = ((const cint*)(uintptr_t)a.ctx)[s];
  } else {
    const cint* ck = (const cint*)(uintptr_t)a.cu_k;
    lk = ck[s + 1] - ck[s];
  }
  r.Lk = min(max(lk, 0), a.capacity);
  return r;
}

// The keys [0, end) that query q, and rows up to `row`, see.
template <bool CAUSAL> __device__ __forceinline__ int sees(const Seq& s, int q) {
  return CAUSAL ? max(q + 1 + (s.Lk - s.Lq), 0) : s.Lk;
}
template <bool CAUSAL> __device__ __forceinline__ int end_of(const Args& a, const Seq& s, int row) {
  return CAUSAL ? sees<CAUSAL>(s, row / a.group) : s.Lk;
}

// Query and head of the group of a row x past row (q, g); x below 2^14.
struct RowAt {
  int q, g;
};
__device__ __forceinline__ RowAt row_past(const Args& a, RowAt r, int x) {
  // y / group as (2 y) * ceil(2^31 / group) >> 32, exact for y, group < 2^15
  const u32 y = (u32)(r.g + x), d = __umulhi(2 * y, a.group31);
  return {r.q + (int)d, (int)(y - d * (u32)a.group)};
}

typedef __attribute__((address_space(3))) unsigned char lds_u8;
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

// 1 KiB straight into LDS (dst + 16 lane); inline assembly, so that the compiler neither
// counts it nor guards LDS reads with waits for it: the waits are explicit.  M0 is used
// by nothing else here.  (s_nop 4: should a vector instruction, such as the restoring of a
// spilled register, have written the resource right before, the load may read it.)
__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t r, int voff, u32 dst) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :
               : "v"(voff), "s"(r), "s"(dst)
               : "memory", "m0");
#pragma clang diagnostic pop
}
__device__ __forceinline__ void load_lds16(const u16* p, u32 dst) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :
               : "v"(p), "s"(dst)
               : "memory", "m0");
#pragma clang diagnostic pop
}

// 0x8000 in each half of x that holds a finite value: with the exponent's bits turned over,
// all of them set leaves 0, which alone stays below 0x8000 when 0x7fff is added.
template <bool F16> __device__ __forceinline__ u32 finite16(u32 x) {
  constexpr u32 kExp = F16 ? 0x7c007c00u : 0x7f807f80u;
  return ((~x & kExp) + 0x7fff7fffu) & 0x80008000u;
}
// 0x8000 -> 0xffff, 0 -> 0 in each half
__device__ __forceinline__ u32 spread16(u32 t) { return (t - (t >> 15)) | t; }

// min(max(end - key, 0), 16) in scalar registers, where the compiler would take a vector
// instruction for the clamp and the buffer resource could not be built.
__device__ __forceinline__ int rows_left(int end, int key) {
  int n;
  asm("s_sub_i32 %0, %1, %2\n\ts_max_i32 %0, %0, 0\n\ts_min_i32 %0, %0, 16" : "=&s"(n) : "s"(end), "s"(key) : "scc");
  return n;
}

// At most N of this wave's loads are in flight and its LDS reads are done, then the
// workgroup's.
template <int N> __device__ __forceinline__ void landed_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// R row blocks of 32 rows, SL key slices of KT sub-tiles an iteration, STAGES of LDS.
template <int R_, int SL_, int KT_, int STAGES_> struct Shape {
  static constexpr int R = R_, SL = SL_, KT = KT_, STAGES = STAGES_;
  static constexpr int kWaves = R * SL, kThreads = 64 * kWaves;
  static constexpr int kKeys = 32 * SL * KT;             // of an iteration
  static constexpr int kTile = SL * KT * kSubBytes;      // bytes of K (or V) of a stage
  static constexpr int kStage = 2 * kTile;
  static constexpr int kGroups = 2 * kKeys / 16 / kWaves;  // 16-row loads a wave brings
  static constexpr int kLoads = 4 * kGroups;             // instructions a wave and stage
  static constexpr int kPart = SL > 1 ? kWaves * 4 * 4096 : 0;  // partial O of the merge
  static constexpr int kOut = kWaves * 32 * kOutPitch;
  static constexpr int kMl = kWaves * 32 * 8;
  static constexpr int kRing = STAGES * kStage;
  // Q comes in through the last stages; those before them are filled at the start
  static constexpr int kQ = kWaves * 8192, kEarly = (kRing - kQ) / kStage;
  static constexpr int kBody = kRing > kPart + kMl ? kRing : kPart + kMl;
  static constexpr int kLds = kBody > kOut ? kBody : kOut;
  static_assert(2 * kKeys % (16 * kWaves) == 0 && kRing >= kQ + kStage && kEarly < STAGES && STAGES - kEarly <= 2, "the form");
  static constexpr int kRows = 32 * R;
  // shared work, in iterations: what an item's start, merge and output cost, and the
  // least a workgroup takes
  static constexpr int kStart = R == 8 ? 2 : 3, kLeast = 6;
};

// Shared work.  Where the items (row block, sequence, KV head) are few or uneven, the
// workgroups of a head divide its iterations evenly instead: the items' iterations, with
// kStart more for each, follow each other on a line, cut into equal shares.  A share is
// the end of one item, whole items, and the start of another; an item that is cut leaves
// partial results, which a second kernel joins in the order of the line.
constexpr int kMaxSharedSeqs = 1024;

struct Line {  // of one KV head: pre[s] is where sequence s begins
  int total, share;
};
struct Item {
  int sg, row0, end, n_it;  // sequence, first row, keys its rows see, iterations of them
  int begin, units;         // its place on the line
  Seq sq;
  int rows;
};

template <class S, bool CAUSAL> __device__ __forceinline__ int units_of(const Args& a, const Seq& sq, int& per) {
  const int rows = sq.rows(a);
  // (the row block with the most keys stands for all of its sequence)
  per = (rows > 0 ? (end_of<CAUSAL>(a, sq, rows - 1) + S::kKeys - 1) / S::kKeys : 0) + S::kStart;
  return min((rows + S::kRows - 1) / S::kRows, a.n_rb) * per;
}

// pre[0 .. n_seqs] in LDS, by NT threads; tmp: one value a wave.
template <class S, bool CAUSAL, int NT>
__device__ __forceinline__ Line line_of(const Args& a, int* pre, int* tmp, int n_shares) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int each = (a.n_seqs + NT - 1) / NT, s0 = min(tid * each, a.n_seqs), s1 = min(s0 + each, a.n_seqs);
  int sum = 0, per;
  for (int s = s0; s < s1; ++s) sum += units_of<S, CAUSAL>(a, seq_of(a, s), per);
  int upto = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(upto, o);
    upto += lane >= o ? x : 0;
  }
  if (lane == 63) tmp[wave] = upto;
  __syncthreads();
  int at = upto - sum;
  for (int w = 0; w < wave; ++w) at += tmp[w];
  for (int s = s0; s < s1; ++s) {
    pre[s] = at;
    at += units_of<S, CAUSAL>(a, seq_of(a, s), per);
  }
  if (tid == NT - 1) pre[a.n_seqs] = at;
  __syncthreads();
  Line l;
  l.total = __builtin_amdgcn_readfirstlane(pre[a.n_seqs]);
  l.share = max((l.total + n_shares - 1) / n_shares, S::kLeast);
  return l;
}

// The item at unit u of the line, u < total.
template <class S, bool CAUSAL> __device__ __forceinline__ Item item_at(const Args& a, const int* pre, int u) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = a.n_seqs;
  while (n > 1) {  // the last s with pre[s] <= u, 64 bounds a step
    const int step = (n + 63) / 64, at = lane * step;
    const int hits = __popcll(__ballot(at < n && pre[lo + min(at, n - 1)] <= u));
    lo += (hits - 1) * step;
    n = min(step, n - (hits - 1) * step);
  }
  Item it;
  it.sg = __builtin_amdgcn_readfirstlane(lo);
  const int begin = __builtin_amdgcn_readfirstlane(pre[lo]);
  it.sq = seq_of(a, it.sg);
  it.rows = it.sq.rows(a);
  const int nrb = min((it.rows + S::kRows - 1) / S::kRows, a.n_rb);
  units_of<S, CAUSAL>(a, it.sq, it.units);
  const int z = (u - begin) / it.units;
  it.begin = begin + z * it.units;
  // causal row blocks: the ones with most and least keys in turn
  it.row0 = (z & 1 ? z >> 1 : nrb - 1 - (z >> 1)) * S::kRows;
  it.end = __builtin_amdgcn_readfirstlane(end_of<CAUSAL>(a, it.sq, min(it.row0 + S::kRows, it.rows) - 1));
  it.n_it = (it.end + S::kKeys - 1) / S::kKeys;
  return it;
}
// Units [x0, x1) of an item as its iterations.
template <class S> __device__ __forceinline__ int iteration_of(const Item& it, int x) {
  return min(max(x - S::kStart, 0), it.n_it);
}

template <class S, bool CAUSAL, bool F16, bool PAGE16, bool SHARED>
__global__ __launch_bounds__(S::kThreads, S::kWaves == 8 ? 2 : 1) void prefill_paged_kernel(Args a) {
  typedef pf::Mfma<F16> M;
  constexpr int SL = S::SL, KT = S::KT, STAGES = S::STAGES, kRows = S::kRows;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[S::kLds];
  __shared__ int pre[SHARED ? kMaxSharedSeqs + 1 + S::kWaves : 1];
  const u32 lds0 = (u32)(uintptr_t)(lds_u8*)lds;

  const int tid = threadIdx.x;

  // KV head fastest: one XCD per head when there are eight
  const int h = blockIdx.x % a.hkv;
  Item item;
  int unit = 0, unit_end = 0;
  if constexpr (SHARED) {
    const Line l = line_of<S, CAUSAL, S::kThreads>(a, pre, pre + kMaxSharedSeqs + 1, gridDim.x / a.hkv);
    unit = (int)(blockIdx.x / a.hkv) * l.share;
    unit_end = min(unit + l.share, l.total);
    // for the joining kernel: whether the share starts inside an item
    Cut cut = {0, -1};
    if (unit >= unit_end) {  // workgroup-uniform
      if (tid == 0) a.ws_cut[blockIdx.x] = cut;
      return;
    }
    item = item_at<S, CAUSAL>(a, pre, unit);
    const int x = unit - item.begin;
    if (x > 0 && x <= l.share) {  // the item's first cut
      const int w = (int)(blockIdx.x / a.hkv);
      // the shares that hold iterations of it: all but perhaps those at its ends
      cut.first = iteration_of<S>(item, x) > 0 ? w - 1 : w;
      cut.last = w - 1;
      for (int k = w; iteration_of<S>(item, k * l.share - item.begin) < item.n_it; ++k) cut.last = k;
      cut.opens = w - 1;
      cut.row0 = item.row0;
      cut.rows = item.rows;
      cut.q_beg = item.sq.q_beg;
    }
    if (tid == 0) a.ws_cut[blockIdx.x] = cut;
  } else {
    // an item a workgroup: the row blocks of a sequence together, the causal ones with
    // the most keys first
    const int i = blockIdx.x / a.hkv, z = i % a.n_rb;
    item.sg = i / a.n_rb;
    item.sq = seq_of(a, item.sg);
    item.rows = item.sq.rows(a);
    const int nrb = min((item.rows + kRows - 1) / kRows, a.n_rb);
    if (z >= nrb) return;  // workgroup-uniform
    item.row0 = (nrb - 1 - z) * kRows;
    item.end = __builtin_amdgcn_readfirstlane(end_of<CAUSAL>(a, item.sq, min(item.row0 + kRows, item.rows) - 1));
    item.n_it = (item.end + S::kKeys - 1) / S::kKeys;
  }
  auto next_item = [&]() {
    if (unit >= unit_end) return false;
    item = item_at<S, CAUSAL>(a, pre, unit);
    return true;
  };
  for (bool more = true; more; more = SHARED && next_item()) {
  // (opaque: else what hangs on them alone is kept from item to item, and registers spill)
  int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if constexpr (SHARED) {
    asm volatile("" : "+v"(lane));
    asm volatile("" : "+s"(wave));
  }
  const int col = lane & 31, hl = lane >> 5;
  const int rb_w = wave % S::R, sl = wave / S::R;  // row block of the workgroup, key slice
  int i0 = 0, i1, slot = -1;  // iterations, place of a partial result
  if constexpr (SHARED) {
    const int x0 = unit - item.begin, x1 = min(item.units, unit_end - item.begin);
    unit = item.begin + x1;
    i0 = __builtin_amdgcn_readfirstlane(iteration_of<S>(item, x0));
    i1 = __builtin_amdgcn_readfirstlane(iteration_of<S>(item, x1));
    // no iteration here (an item of none at all: its zeros are the first share's)
    if (item.n_it == 0 ? x0 > 0 : i0 == i1) continue;
    // cut: only a share's first item can have begun before it, only its last go on
    if (i1 - i0 < item.n_it) slot = 2 * (int)blockIdx.x + (x0 > 0 ? 0 : 1);
  } else {
    i1 = item.n_it;
  }
  const Seq& sq = item.sq;
  const int sg = item.sg, rows = item.rows, row0 = item.row0, kv_end = item.end;
  // sub-tiles [j0, j1) of 32 keys
  const int j0 = i0 * SL * KT, j1 = min(i1 * SL * KT, (kv_end + 31) / 32);
  const int n_it = i1 - i0;

  // this wave's and lane's rows
  const int wrow = row0 + 32 * rb_w;
  const int w_row = min(wrow, rows - 1), w_last = rows - 1 - w_row;  // (a wave past the rows: the last one)
  RowAt w_at;
  w_at.q = __builtin_amdgcn_readfirstlane(w_row / a.group);
  w_at.g = w_row - w_at.q * a.group;
  const int my_q = row_past(a, w_at, min(col, w_last)).q;
  const int w_end = wrow < rows ? end_of<CAUSAL>(a, sq, min(wrow + 31, rows - 1)) : 0;
  const int full = sees<CAUSAL>(sq, w_at.q);  // keys below need no mask
  const int my_lim = sees<CAUSAL>(sq, my_q);
  const int w_sub = min(j1, (w_end + 31) / 32);

  // ---- staging: 16-row group g of a stage is rows 16 g of K, then of V; this wave's
  // are wave * kGroups and up.  16-byte chunk ch of row r sits at ch ^ (r & 15) (K) or
  // ch ^ 4 (r & 3) (V).
  typedef const int32_t __attribute__((address_space(4))) cint;
  const cint* tab = (const cint*)(uintptr_t)(a.tables + (int64_t)sg * a.max_blocks);
  constexpr int kKGroups = S::kKeys / 16;
  const int r4 = lane >> 4;
  int voff_k[4], voff_v;  // (rows of i = 1..3 of V: 4 i rows further)
#pragma unroll
  for (int i = 0; i < 4; ++i) voff_k[i] = (4 * i + r4) * a.row_bytes + 16 * ((lane & 15) ^ (4 * i + r4));
  voff_v = r4 * a.row_bytes + 16 * ((lane & 15) ^ (4 * r4));
  const int key_base = 32 * j0;
  int ent[S::kGroups];  // block numbers of the next stage's groups
  auto first_key = [&](int n, int gi) { return key_base + n * S::kKeys + 16 * ((wave * S::kGroups + gi) % kKGroups); };
  auto look_up = [&](int n, int* ent) {
    if constexpr (PAGE16) {
#pragma unroll
      for (int gi = 0; gi < S::kGroups; ++gi)
        ent[gi] = tab[min(divide(a, first_key(n, gi) >> 4), a.max_blocks - 1)];
    }
  };
  auto issue = [&](int n, const int* ent) {
    const u32 st = lds0 + (u32)(n % STAGES * S::kStage);
#pragma unroll
    for (int gi = 0; gi < S::kGroups; ++gi) {
      const int g = wave * S::kGroups + gi;
      const bool is_k = g < kKGroups;
      const int key = first_key(n, gi);
      const u16* cache = (is_k ? a.kc : a.vc) + h * D;
      const u32 dst = st + (u32)(g * 4096);
      if constexpr (PAGE16) {
        const int page = divide(a, key >> 4);
        const int64_t blk = (u32)ent[gi] < a.num_blocks ? ent[gi] : 0;
        const int64_t row = blk * a.block_size + (key - page * a.block_size);
        // (the head's 256 bytes of a row lie before the next row's)
        const int n_rows = rows_left(kv_end, key);
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<u16*>(cache + row * (u32)(a.row_bytes >> 1)), 0, n_rows * a.row_bytes, 0x00020000);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          load_lds16(rs, is_k ? voff_k[i] : voff_v + 4 * i * a.row_bytes, dst + i * 1024);
      } else {
        // every lane's own row; rows behind the context repeat its last one (masked)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 4 * i + r4;
          const int k = min(key + r, kv_end - 1);
          const int page = divide(a, k);
          const int e = a.tables[(int64_t)sg * a.max_blocks + page];
          const int64_t blk = (u32)e < a.num_blocks ? e : 0;
          const int64_t row = blk * a.block_size + (k - page * a.block_size);
          const int ch = (lane & 15) ^ (is_k ? r : 4 * r4);
          load_lds16(cache + row * (a.row_bytes >> 1) + 8 * ch, dst + i * 1024);
        }
      }
    }
  };
  // ---- on their way: this wave's rows of Q, into its place in the last stages (chunks
  // swizzled as K's), then the first stages: all their block numbers, then all their rows
  const u32 q_lds = lds0 + (u32)(S::kRing - S::kQ + wave * 8192);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + r4;
    const RowAt at = row_past(a, w_at, min(r, w_last));
    load_lds16(a.q + (int64_t)(sq.q_beg + at.q) * a.q_stride + (h * a.group + at.g) * D + 8 * ((lane & 15) ^ (r & 15)),
               q_lds + i * 1024);
  }
  {
    int first[S::kEarly][S::kGroups];
#pragma unroll
    for (int n = 0; n < S::kEarly; ++n) look_up(n, first[n]);
#pragma unroll
    for (int n = 0; n < S::kEarly; ++n)
      if (n < n_it) issue(n, first[n]);
  }
  int late[STAGES - S::kEarly][S::kGroups];  // of those that go out once Q has been read
#pragma unroll
  for (int n = S::kEarly; n < STAGES; ++n) look_up(n, late[n - S::kEarly]);

  // fragment addresses within a sub-tile (see prefill_wide.hip)
  int koff[8], vo[4];
#pragma unroll
  for (int t = 0; t < 8; ++t) koff[t] = col * 256 + 16 * ((2 * t + hl) ^ (col & 15));
  {
    const int g = lane >> 4, i = lane & 15;
    const int l0 = (4 * (g >> 1) + (i >> 2)) * 256 + 32 * (g & 1) + 8 * (i & 3);
#pragma unroll
    for (int db = 0; db < 4; ++db) vo[db] = l0 + 64 * (db ^ (i >> 2));
  }

  const float cs = a.scale_log2, kthr = kRescale / cs;
  f32x16 o[4];
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  float m = -1e30f, l = 0.f;  // reference max (raw scores), lane-partial row sum

  f32x16 s;      // scores of a sub-tile, then:
  u32x4 pb[2];   // its probabilities, two steps of 16 keys
  u32x4 qf[8], kf[8], vf[8];
  typedef const __attribute__((address_space(3))) u32x4 lds_u32x4;
  auto tile = [&](int n, int sub) { return (const lds_u8*)lds + n % STAGES * S::kStage + sub * kSubBytes; };
  auto read_k = [&](const lds_u8* kb) {
#pragma unroll
    for (int t = 0; t < 8; ++t) kf[t] = *reinterpret_cast<lds_u32x4*>(kb + koff[t]);
  };
  auto v_frag = [&](const lds_u8* vb, int i) {  // step i / 4, dims 32 (i % 4) and up
    const lds_u8* at = vb + vo[i & 3] + 4096 * (i >> 2);
    const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at);
    const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 2048));
    const u32x2 a0 = __builtin_bit_cast(u32x2, lo), a1 = __builtin_bit_cast(u32x2, hi);
    return u32x4{a0[0], a0[1], a1[0], a1[1]};
  };
  auto read_v = [&](const lds_u8* vb) {
#pragma unroll
    for (int i = 0; i < 8; ++i) vf[i] = v_frag(vb, i);
  };
  auto scores = [&]() {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int t = 0; t < 8; ++t) s = M::run(kf[t], qf[t], s);
  };
  auto product = [&]() {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i & 3] = M::run(vf[i], pb[i >> 2], o[i & 3]);
  };
  // Probabilities of sub-tile j's scores; its values are at vb, their fragments in vf.
  auto softmax = [&](int j, const lds_u8* vb) {
    const bool masked = 32 * j + 32 > full;
    if (masked) {
      const int lim = my_lim - 32 * j - 4 * hl;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 8 * (i >> 2) + (i & 3) < lim ? s[i] : -INFINITY;
    }
    float mx = vmax3(s[0], s[1], s[2]);
#pragma unroll
    for (int i = 3; i < 15; i += 2) mx = vmax3(mx, s[i], s[i + 1]);
    mx = vmax(mx, s[15]);
    if (__ballot(!(mx <= m + kthr))) {  // any lane (or a NaN): rescale (rare after the first sub-tile)
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
      mx = vmax(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
      // (only the rows that need it: a row's result does not hang on its neighbours)
      const float mn = mx <= m + kthr ? m : vmax(m, mx), alpha = fast_exp2((m - mn) * cs);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
    }
    const float nb = -m * cs;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const u32 p = M::pack(fast_exp2(fmaf(s[2 * w], cs, nb)), fast_exp2(fmaf(s[2 * w + 1], cs, nb)));
      pb[w >> 2][w & 3] = p;
      l = M::dot2_ones(p, l);
    }
    if (masked) {
      // A value that a row does not see must not reach it, whatever it is: with an
      // infinity or a NaN among these 32 keys' values, the product takes 0 in its place
      // and the rows that see its key add it
      u32 fine = 0x80008000u;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) fine &= finite16<F16>(vf[i][e]);
      if (__ballot(fine != 0x80008000u)) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) vf[i][e] &= spread16(finite16<F16>(vf[i][e]));
        const int seen = my_lim - 32 * j;
#pragma unroll 1
        for (int k = 0; k < 32; ++k) {
          const u32 on = k < seen ? ~0u : 0u;
#pragma unroll
          for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              // dims 32 db + 8 r + 4 hl .. + 3 of key k; the finite ones add 0
              const u32x2 x = *reinterpret_cast<const __attribute__((address_space(3))) u32x2*>(
                  vb + k * 256 + 16 * ((4 * db + r) ^ (4 * (k & 3))) + 8 * hl);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const u32 y = x[e] & ~spread16(finite16<F16>(x[e])) & on;
                o[db][4 * r + 2 * e] += F16 ? f16lo(y) : bf16lo(y);
                o[db][4 * r + 2 * e + 1] += F16 ? f16hi(y) : bf16hi(y);
              }
            }
        }
      }
    }
  };

  // Q fragments (B operand of S^T = K Q^T: lane = row), once the wave's own loads of them,
  // the oldest, have landed
  if (n_it >= S::kEarly) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(S::kEarly * S::kLoads) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
  for (int t = 0; t < 8; ++t) qf[t] = *reinterpret_cast<lds_u32x4*>((const lds_u8*)lds + (q_lds - lds0) + koff[t]);

  // stage 0 has landed and every wave is done with Q
  if (S::kEarly > 1 && n_it >= S::kEarly) landed_barrier<(S::kEarly - 1) * S::kLoads>();
  else landed_barrier<0>();
#pragma unroll
  for (int k = S::kEarly; k < STAGES; ++k)
    if (k < n_it) issue(k, late[k - S::kEarly]);
  look_up(STAGES, ent);

  for (int n = 0; n < n_it; ++n) {
    if (n > 0) {
      // stage n has landed and every wave is done with stage n - 1
      if (STAGES > 2 && n + STAGES - 2 < n_it) landed_barrier<(STAGES - 2) * S::kLoads>();
      else landed_barrier<0>();
      if (n + STAGES - 1 < n_it) {
        issue(n + STAGES - 1, ent);
        look_up(n + STAGES, ent);
      }
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int j = j0 + (n * SL + sl) * KT + kt;
      if (j >= w_sub) break;  // wave-uniform
      const lds_u8* kb = tile(n, sl * KT + kt);
      read_k(kb);
      scores();
      read_v(kb + S::kTile);
      softmax(j, kb + S::kTile);
      product();
    }
  }

  // ---- merge the slices of each row block: slice s takes dims 128 s / SL and up, its own
  // part from registers, the others' through LDS (over the dead stages)
  {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
  __syncthreads();
  float mt = m, lt = l;
  if constexpr (SL > 1) {
    auto part = [&](int w, int db) { return reinterpret_cast<f32x4*>(lds + (4 * w + db) * 4096); };
    float2* ml = reinterpret_cast<float2*>(lds + S::kPart);
    if (lane < 32) ml[wave * 32 + col] = make_float2(m, l);
#pragma unroll
    for (int db = 0; db < 4; ++db)
      if (db * SL / 4 != sl) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          part(wave, db)[r * 64 + lane] = f32x4{o[db][4 * r], o[db][4 * r + 1], o[db][4 * r + 2], o[db][4 * r + 3]};
      }
    __syncthreads();
    float2 mls[SL];
    mt = -1e30f;
#pragma unroll
    for (int k = 0; k < SL; ++k) {
      mls[k] = ml[(k * S::R + rb_w) * 32 + col];
      mt = vmax(mt, mls[k].x);
    }
    float wt[SL];
    lt = 0.f;
#pragma unroll
    for (int k = 0; k < SL; ++k) {
      wt[k] = fast_exp2((mls[k].x - mt) * cs);
      lt = fmaf(mls[k].y, wt[k], lt);
    }
#pragma unroll
    for (int db = 0; db < 4; ++db)
      if (db * SL / 4 == sl) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < SL; ++k) {  // in slice order
            if (k == db * SL / 4) {
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = fmaf(o[db][4 * r + e], wt[k], v[e]);
            } else {
              const f32x4 x = part(k * S::R + rb_w, db)[r * 64 + lane];
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = fmaf(x[e], wt[k], v[e]);
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) o[db][4 * r + e] = v[e];
        }
      }
  }

  if (slot >= 0) {  // a part of the item: unnormalised, in fp32, as the lanes hold it
    const int at = slot * S::R + rb_w;
    if (sl == 0 && hl == 0) a.ws_ml[(int64_t)at * 32 + col] = make_float2(mt * cs, lt);
    f32x4* dst = reinterpret_cast<f32x4*>(a.ws_o) + (int64_t)at * 1024 + lane;
#pragma unroll
    for (int db = 0; db < 4; ++db)
      if (SL == 1 || db * SL / 4 == sl) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          dst[(4 * db + r) * 64] = f32x4{o[db][4 * r], o[db][4 * r + 1], o[db][4 * r + 2], o[db][4 * r + 3]};
      }
    __syncthreads();  // the next item's loads overwrite what the merge read
    continue;
  }
  const float inv = lt > 0.f ? __builtin_amdgcn_rcpf(lt) : (lt == 0.f ? 0.f : lt);  // (a NaN stays one)
  if constexpr (SL > 1) __syncthreads();  // the partial results have been read
  unsigned char* stg = lds + rb_w * (32 * kOutPitch);
#pragma unroll
  for (int db = 0; db < 4; ++db)
    if (SL == 1 || db * SL / 4 == sl) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        u32x2 w;
        w[0] = M::pack(o[db][4 * r] * inv, o[db][4 * r + 1] * inv);
        w[1] = M::pack(o[db][4 * r + 2] * inv, o[db][4 * r + 3] * inv);
        *reinterpret_cast<u32x2*>(stg + col * kOutPitch + (32 * db + 8 * r + 4 * hl) * 2) = w;
      }
    }
  __syncthreads();
  // whole rows: 16 lanes a row
  RowAt at0;
  at0.q = __builtin_amdgcn_readfirstlane(row0 / a.group);
  at0.g = row0 - at0.q * a.group;
  for (int r = tid >> 4; r < min(kRows, rows - row0); r += S::kThreads / 16) {
    const RowAt at = row_past(a, at0, r);
    *reinterpret_cast<u32x4*>(a.out + (int64_t)(sq.q_beg + at.q) * a.o_stride + (h * a.group + at.g) * D + (lane & 15) * 8) =
        *reinterpret_cast<const u32x4*>(lds + (r >> 5) * (32 * kOutPitch) + (r & 31) * kOutPitch + (lane & 15) * 16);
  }
  if constexpr (!SHARED) break;
  __syncthreads();
  }
}

// Joins the parts of a cut item, in the line's order: workgroup (x, y) those of cut x, row
// block y of 32, a wave 32 dims, in the layout the parts' waves left them.
template <class S, bool F16>
__global__ __launch_bounds__(256) void prefill_paged_join_kernel(Args a) {
  const Cut c = a.ws_cut[blockIdx.x + a.hkv];  // (share 0 of a head begins no cut)
  const int h = blockIdx.x % a.hkv, rb = blockIdx.y, lane = threadIdx.x & 63, hl = lane >> 5, col = lane & 31;
  if (c.first >= c.last || c.row0 + 32 * rb >= c.rows) return;
  const int db = threadIdx.x >> 6;
  auto place_of = [&](int w) { return (int64_t)(2 * (w * a.hkv + h) + (w == c.opens ? 1 : 0)) * S::R + rb; };
  float mx = -3e38f, lt = 0.f;
#pragma unroll 4
  for (int w = c.first; w <= c.last; ++w) mx = vmax(mx, a.ws_ml[place_of(w) * 32 + col].x);
  f32x4 acc[4] = {};
#pragma unroll 2
  for (int w = c.first; w <= c.last; ++w) {
    const int64_t at = place_of(w);
    const float2 ml = a.ws_ml[at * 32 + col];
    const f32x4* src = reinterpret_cast<const f32x4*>(a.ws_o) + at * 1024 + 256 * db + lane;
    const float wt = fast_exp2(ml.x - mx);
    lt = fmaf(ml.y, wt, lt);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const f32x4 v = src[64 * r];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[r][e] = fmaf(v[e], wt, acc[r][e]);
    }
  }
  const int row = c.row0 + 32 * rb + col;
  if (row >= c.rows) return;
  const float inv = lt > 0.f ? __builtin_amdgcn_rcpf(lt) : (lt == 0.f ? 0.f : lt);
  const int qi = row / a.group, head = h * a.group + row - qi * a.group;
  u16* out = a.out + (int64_t)(c.q_beg + qi) * a.o_stride + head * D + 32 * db + 4 * hl;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    u32x2 w;
    w[0] = pf::Mfma<F16>::pack(acc[r][0] * inv, acc[r][1] * inv);
    w[1] = pf::Mfma<F16>::pack(acc[r][2] * inv, acc[r][3] * inv);
    *reinterpret_cast<u32x2*>(out + 8 * r) = w;
  }
}

// ------------------------------------------------------------------ host
typedef Shape<2, 4, 1, 2> Rows64;
typedef Shape<4, 2, 1, 4> Rows128;
typedef Shape<8, 1, 2, 4> Rows256;

struct Plan {
  int rows;    // of a workgroup: 64, 128 or 256
  int shares;  // of a KV head's work, or 0: an item a workgroup
  size_t bytes;
};

static Plan plan(int32_t n_seqs, int32_t max_q, int32_t max_k, int64_t cap, int32_t hq, int32_t hkv, int n_cu) {
  Plan p = {};
  // (every sequence is counted as long as the longest: of single tokens beside a long chunk the
  // items are far fewer than this says)
  const int64_t rows = (int64_t)max_q * (hq / hkv);
  auto items_of = [&](int r) { return (int64_t)n_seqs * hkv * cdiv(rows, r); };
  // Rows of a workgroup, us in 64 / 128 / 256 of them.  Where one block holds a sequence's
  // rows the keys are what it costs: 16 x 5 queries over 1.5k keys at 16/8 heads 22.9 / 29.5
  // / 31.1, 64 x 4 over 4k at 32/8 190 / 183 / 187.  Short contexts of few items are a chain
  // of latencies, shortest in small blocks that do not outnumber the CUs: 1 x 97 over 98
  // 7.6 / 8.3 / 9.2, 11 x 64 over 171 at 32/8 16.3 / 10.2 / 12.0, 6 x 306 at 32/8 32 / 22.5
  // / 17.5; at one iteration of 64 keys in the large ones, which have no key slices to
  // merge: 13 x 8 7.1 / 6.8 / 6.2, 28 x 42 13.1 / 7.9 / 7.3.  Else every key a workgroup
  // brings in serves more rows in large ones: 2 x 265 over 8.9k at 64/8 250 / 205 / 180,
  // 26 x 1301 over 1.8k 584 / 430 / 380.
  if (max_k <= 64) p.rows = 256;
  else if (rows <= 64) p.rows = items_of(64) < n_cu ? 64 : 128;
  else if (max_k <= 1024 && items_of(64) <= n_cu) p.rows = 64;
  else if (rows <= 128 || (max_k <= 1024 && items_of(128) <= n_cu)) p.rows = 128;
  else p.rows = 256;
  const int64_t items = items_of(p.rows);
  const int64_t keys = p.rows == 64 ? 128 : 64, its = cdiv(max_k, keys), start = p.rows == 256 ? 2 : 3;
  // In iterations of a workgroup, if all sequences were as long as the longest: an item a
  // workgroup takes whole rounds of the longest; shared work its even part, and some 8
  // for finding it and joining.  (Uneven sequences only make the first worse.)
  const int64_t alone = cdiv(items, n_cu) * (its + start), shared = items * (its + 2 * start) / n_cu + 8;
  // units of a line below 2^30
  const bool fits = n_seqs <= kMaxSharedSeqs && hkv <= n_cu &&
                    cdiv(rows, p.rows) * n_seqs * (cdiv(cap, keys) + start) < (int64_t(1) << 30);
  if (fits && items < 8 * (int64_t)n_cu && 20 * shared < 21 * alone) {
    p.shares = n_cu / hkv;
    p.bytes = (size_t)p.shares * hkv * (2 * p.rows * (D * 4 + 8) + sizeof(Cut));
  }
  return p;
}

template <class S, bool CAUSAL, bool F16>
static int launch_s(Args a, const Plan& p, bool page16, int32_t max_q, hipStream_t st) {
  a.n_rb = (int)cdiv((int64_t)max_q * a.group, S::kRows);
  const dim3 block(S::kThreads);
  if (p.shares) {
    const unsigned grid = (unsigned)p.shares * a.hkv;
    a.ws_ml = (float2*)(a.ws_o + (size_t)grid * 2 * S::kRows * D);
    a.ws_cut = (Cut*)(a.ws_ml + (size_t)grid * 2 * S::kRows);
    if (page16) hipLaunchKernelGGL((prefill_paged_kernel<S, CAUSAL, F16, true, true>), dim3(grid), block, 0, st, a);
    else hipLaunchKernelGGL((prefill_paged_kernel<S, CAUSAL, F16, false, true>), dim3(grid), block, 0, st, a);
    if (p.shares > 1)
      hipLaunchKernelGGL((prefill_paged_join_kernel<S, F16>),
                         dim3((unsigned)(p.shares - 1) * a.hkv, S::R), dim3(256), 0, st, a);
    return AAC_OK;
  }
  // A launch numbers its threads in 32 bits.  One holds whole sequences, each taken to be as
  // long as the longest: where they are too many the next launch takes the others.
  const int64_t of_seq = (int64_t)a.n_rb * a.hkv, most = ((int64_t(1) << 32) - 1) / S::kThreads;
  if (of_seq > most) return AAC_ERR_UNSUPPORTED;  // (one sequence: its queries alone hold 512 GiB)
  for (int64_t left = a.n_seqs; left > 0;) {
    a.n_seqs = (int32_t)std::min(left, most / of_seq);
    const dim3 grid((unsigned)(a.n_seqs * of_seq));
    if (page16) hipLaunchKernelGGL((prefill_paged_kernel<S, CAUSAL, F16, true, false>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((prefill_paged_kernel<S, CAUSAL, F16, false, false>), grid, block, 0, st, a);
    left -= a.n_seqs;
    if (a.cu_q) {
      a.cu_q += a.n_seqs;
    } else {
      a.q += a.n_seqs * a.max_q * a.q_stride;
      a.out += a.n_seqs * a.max_q * a.o_stride;
    }
    if (a.ctx) a.ctx += a.n_seqs;
    else a.cu_k += a.n_seqs;
    a.tables += (int64_t)a.n_seqs * a.max_blocks;
  }
  return AAC_OK;
}

template <bool CAUSAL, bool F16>
static int launch_r(const Args& a, const Plan& p, bool page16, int32_t max_q, hipStream_t st) {
  switch (p.rows) {
    case 64: return launch_s<Rows64, CAUSAL, F16>(a, p, page16, max_q, st);
    case 128: return launch_s<Rows128, CAUSAL, F16>(a, p, page16, max_q, st);
    default: return launch_s<Rows256, CAUSAL, F16>(a, p, page16, max_q, st);
  }
}

}  // namespace pp
}  // namespace aac

using namespace aac;

// The longest context the work is split for: the caller's estimate within what a table
// can name.
static int64_t capacity_of(int32_t block_size, int32_t max_blocks) {
  return std::min<int64_t>((int64_t)max_blocks * block_size, (int64_t(1) << 31) - 4096);
}
static int32_t longest_of(int32_t max_context_len, int64_t cap) {
  return max_context_len > 0 ? (int32_t)std::min<int64_t>(max_context_len, cap) : (int32_t)cap;
}

extern "C" size_t aac_prefill_paged_workspace_bytes(int64_t n_tokens, int32_t n_seqs, int32_t max_seqlen_q,
                                                    int32_t max_context_len, int32_t block_size,
                                                    int32_t max_blocks_per_seq, int32_t n_q_heads,
                                                    int32_t n_kv_heads) {
  int n_cu = 0;
  if (n_tokens <= 0 || n_seqs <= 0 || max_seqlen_q <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 ||
      n_q_heads % n_kv_heads || block_size <= 0 || max_blocks_per_seq <= 0 || device_cu_count(&n_cu) != AAC_OK)
    return 0;
  const int64_t cap = capacity_of(block_size, max_blocks_per_seq);
  return pp::plan(n_seqs, (int32_t)std::min<int64_t>(max_seqlen_q, n_tokens), longest_of(max_context_len, cap), cap,
                  n_q_heads, n_kv_heads, n_cu).bytes;
}

extern "C" int aac_prefill_paged(const void* q, int64_t q_tok_stride, int64_t n_tokens, const void* k_cache,
                                 const void* v_cache, int64_t num_blocks, int32_t block_size,
                                 const int32_t* block_tables, int32_t max_blocks_per_seq,
                                 const int32_t* cu_seqlens_q, const int32_t* context_lens,
                                 const int32_t* cu_seqlens_k, int32_t n_seqs, int32_t max_seqlen_q,
                                 int32_t max_context_len, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                 float scale, int32_t causal, void* out, int64_t out_tok_stride, void* workspace,
                                 size_t workspace_bytes, int32_t dtype, void* stream) {
  if (dtype != AAC_DTYPE_BF16 && dtype != AAC_DTYPE_FP16) return AAC_ERR_UNSUPPORTED;
  if (head_dim != pp::D) return AAC_ERR_UNSUPPORTED;
  if (n_tokens < 0 || n_seqs < 0 || n_q_heads <= 0 || n_kv_heads <= 0 || max_seqlen_q < 0 || num_blocks < 0 ||
      block_size <= 0 || max_blocks_per_seq <= 0 || q_tok_stride < 0 || out_tok_stride < 0 || !(scale > 0.f) ||
      scale > 1e38f)
    return AAC_ERR_INVALID_ARGUMENT;
  if (n_q_heads % n_kv_heads || n_tokens >= (int64_t(1) << 31) ||
      (!cu_seqlens_q && n_tokens != (int64_t)n_seqs * max_seqlen_q))
    return AAC_ERR_SHAPE;
  if (n_tokens == 0 || n_seqs == 0 || max_seqlen_q == 0) return AAC_OK;
  max_seqlen_q = (int32_t)std::min<int64_t>(max_seqlen_q, n_tokens);  // (any bound will do)
  if (!q || !out || !block_tables || (!context_lens && !cu_seqlens_k))
    return AAC_ERR_INVALID_ARGUMENT;
  if (num_blocks == 0 || !k_cache || !v_cache) return AAC_ERR_INVALID_ARGUMENT;
  if (q_tok_stride < (int64_t)n_q_heads * head_dim || out_tok_stride < (int64_t)n_q_heads * head_dim)
    return AAC_ERR_SHAPE;
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) % 16 || q_tok_stride % 8 ||
      out_tok_stride % 8)
    return AAC_ERR_MISALIGNED;
  // 16 rows of the cache, all heads, within a buffer resource's 32-bit offsets; rows of a
  // sequence numbered in int32; positions in 27 bits of groups or rows
  const int64_t cap = capacity_of(block_size, max_blocks_per_seq);
  if ((int64_t)n_kv_heads * head_dim * 2 * 16 >= (int64_t(1) << 31) ||
      (int64_t)max_seqlen_q * (n_q_heads / n_kv_heads) >= (int64_t(1) << 30) || n_q_heads / n_kv_heads >= 1 << 14)
    return AAC_ERR_UNSUPPORTED;
  const bool one = max_blocks_per_seq == 1, page16 = one || block_size % 16 == 0;
  if (!page16 && cap > (int64_t(1) << 27)) return AAC_ERR_UNSUPPORTED;
  pp::Args a = {};
  a.q = (const u16*)q;
  a.kc = (const u16*)k_cache;
  a.vc = (const u16*)v_cache;
  a.out = (u16*)out;
  a.q_stride = q_tok_stride;
  a.o_stride = out_tok_stride;
  a.cu_q = cu_seqlens_q;
  a.ctx = context_lens;
  a.cu_k = cu_seqlens_k;
  a.tables = block_tables;
  a.num_blocks = (u32)std::min<int64_t>(num_blocks, INT32_MAX);
  a.n_tokens = n_tokens;
  a.n_seqs = n_seqs;
  a.hq = n_q_heads;
  a.hkv = n_kv_heads;
  a.group = n_q_heads / n_kv_heads;
  a.group31 = (u32)cdiv(int64_t(1) << 31, a.group);
  a.max_q = max_seqlen_q;
  a.block_size = block_size;
  a.max_blocks = max_blocks_per_seq;
  a.capacity = (int)cap;
  a.row_bytes = n_kv_heads * head_dim * 2;
  a.scale_log2 = scale * kLog2e;
  {
    // a single block: every key is on page 0
    const int64_t d = one ? int64_t(1) << 27 : page16 ? block_size / 16 : block_size;
    u32 s = 0;
    while ((int64_t(1) << s) < d) ++s;
    a.magic = (u32)cdiv(int64_t(1) << (27 + s), d);
    a.shift = 27 + s;
  }
  int n_cu = 0;
  int rc = device_cu_count(&n_cu);
  if (rc != AAC_OK) return rc;
  const pp::Plan p = pp::plan(n_seqs, max_seqlen_q, longest_of(max_context_len, cap), cap, n_q_heads, n_kv_heads, n_cu);
  if (p.bytes) {
    if (!workspace || workspace_bytes < p.bytes) return AAC_ERR_WORKSPACE;
    if ((uintptr_t)workspace % 16) return AAC_ERR_MISALIGNED;
    a.ws_o = (float*)workspace;
  }
  hipStream_t st = (hipStream_t)stream;
  const bool f16 = dtype == AAC_DTYPE_FP16;
  if (causal) rc = f16 ? pp::launch_r<true, true>(a, p, page16, max_seqlen_q, st)
                       : pp::launch_r<true, false>(a, p, page16, max_seqlen_q, st);
  else rc = f16 ? pp::launch_r<false, true>(a, p, page16, max_seqlen_q, st)
                : pp::launch_r<false, false>(a, p, page16, max_seqlen_q, st);
  if (rc != AAC_OK) return rc;
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? AAC_OK : (int)e;
}
