/*
 * aac_attn.h -- C ABI of libaac_attn.so, the MI355X (gfx950) attention hot
 * path of the Qwen3 serving engine: the slot_mapping KV-cache store, varlen
 * causal GQA prefill and paged decode.
 *
 * Conventions shared by every entry point
 *   - All tensor pointers are device pointers; every buffer is owned by the
 *     caller.  The library allocates no device memory (aac_decode_paged_noalloc
 *     uses one static device array instead of a workspace argument).
 *   - `stream` is a hipStream_t passed as void* (NULL = the null stream).
 *     Work is enqueued asynchronously; no entry point synchronises the host.
 *   - Strides are in ELEMENTS.  Within one token the [heads, head_dim] block
 *     must be contiguous (head stride == head_dim, dim stride == 1); only the
 *     token (or sequence) stride is free.  This admits the reference's v,
 *     a strided view of the fused qkv buffer with token stride
 *     (Hq + 2*Hkv) * head_dim (llm.py:156, model/model.py:222).
 *   - Caches are [num_blocks, block_size, n_kv_heads, head_dim], token-major
 *     ("NHD").  The reference's slot cache [num_slots, max_seq_len, Hkv, D]
 *     (model/model.py:324-336) is the case block_size = max_seq_len with one
 *     block per sequence (block_tables[b] = {slot_b}).
 *   - Return value: 0 on success, a negative AAC_ERR_* code for a rejected
 *     argument, or a positive hipError_t when a launch failed.  Nothing is
 *     thrown across the ABI; aac_strerror() gives the message.
 *   - Calls are stateless and reentrant, except aac_decode_paged_noalloc,
 *     whose calls share one scratch array per GPU.
 *
 * Reference interfaces replaced (reference paths are relative to the
 * yijichar/AWesome_ACceleration tree):
 *   aac_kv_store             kv_flat.index_copy_(0, scatter_indices, k)/(v)
 *                            llm.py:171-174
 *   aac_kv_append_paged      the k=/v= append half of flash_attn_with_kvcache
 *                            model/model.py:233-240
 *   aac_prefill_varlen       flash_attn_varlen_func(..., causal=True)
 *                            llm.py:178-184 (also flash_attn_func,
 *                            model/model.py:253-254, with uniform cu_seqlens)
 *   aac_prefill_varlen_store llm.py:171-184 (store + attend in one call)
 *   aac_decode_paged         the attend half of flash_attn_with_kvcache
 *                            model/model.py:233-240
 *   aac_decode_append_paged  all of flash_attn_with_kvcache(k=, v=)
 *                            model/model.py:233-240
 */
#ifndef AAC_ATTN_H
#define AAC_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define AAC_ABI_VERSION 2

/* element types */
enum {
  AAC_DTYPE_BF16 = 0,
  AAC_DTYPE_FP16 = 1,
  AAC_DTYPE_FP32 = 2
};

/* status codes (positive values are hipError_t) */
enum {
  AAC_OK = 0,
  AAC_ERR_INVALID_ARGUMENT = -1, /* null pointer, negative or zero size  */
  AAC_ERR_UNSUPPORTED = -2,      /* dtype / head_dim / GQA group not built */
  AAC_ERR_MISALIGNED = -3,       /* pointer or stride breaks 16-B access  */
  AAC_ERR_WORKSPACE = -4,        /* split-K workspace too small           */
  AAC_ERR_SHAPE = -5,            /* inconsistent shape arguments          */
  AAC_ERR_SCRATCH = -6           /* plan exceeds the static decode scratch */
};

/* ABI revision of the loaded library (AAC_ABI_VERSION it was built with). */
int aac_abi_version(void);

/* Message for a status code returned by any entry point (never NULL). */
const char* aac_strerror(int code);

/*
 * KV store: for t in [0, n_tokens):
 *   if slot_mapping[t] >= 0:
 *     k_cache_rows[slot_mapping[t]] = k[t];  v_cache_rows[slot_mapping[t]] = v[t]
 * where *_cache_rows views the cache as [num_cache_rows, n_kv_heads, head_dim].
 * Byte copy: the cache contents are bit-exact.  A negative slot is padding and
 * is skipped; a slot >= num_cache_rows is skipped too (never written), which the
 * reference would reject with an IndexError -- validate on the host if that
 * matters.  Duplicate slots leave an unspecified one of the rows.
 * Replaces llm.py:171-174.
 */
int aac_kv_store(const void* k, const void* v, int64_t k_tok_stride, int64_t v_tok_stride,
                 void* k_cache, void* v_cache, int64_t num_cache_rows,
                 const int64_t* slot_mapping, int64_t n_tokens, int32_t n_kv_heads,
                 int32_t head_dim, int32_t dtype, void* stream);

/*
 * Decode append: the new token of sequence b (k[b], v[b]) is written at
 * position p = cache_seqlens[b], i.e. cache row
 *   block_tables[b * max_blocks_per_seq + p / block_size] * block_size + p % block_size.
 * cache_seqlens is NOT modified (the reference's caller increments it,
 * model/model.py:241).  Positions beyond the table capacity and block ids
 * outside [0, num_blocks) are skipped.
 * Replaces the k=/v= half of flash_attn_with_kvcache (model/model.py:233-240).
 */
int aac_kv_append_paged(const void* k, const void* v, int64_t k_tok_stride, int64_t v_tok_stride,
                        void* k_cache, void* v_cache, int64_t num_blocks, int32_t block_size,
                        const int32_t* block_tables, int32_t max_blocks_per_seq,
                        const int32_t* cache_seqlens, int32_t n_seqs, int32_t n_kv_heads,
                        int32_t head_dim, int32_t dtype, void* stream);

/*
 * Varlen attention over packed segments.  Segment s owns query rows
 * [cu_seqlens_q[s], cu_seqlens_q[s+1]) and key rows
 * [cu_seqlens_k[s], cu_seqlens_k[s+1]).  Query head h reads KV head
 * h / (n_q_heads / n_kv_heads).  With causal != 0 the mask is bottom-right
 * aligned (query i sees keys j <= i + Lk - Lq); a query row that sees no key
 * gets zeros.  Softmax in fp32, output rounded to dtype.
 *   q   [Nq, n_q_heads, head_dim]  token stride q_tok_stride
 *   k,v [Nk, n_kv_heads, head_dim] token strides k_tok_stride / v_tok_stride
 *   out [Nq, n_q_heads, head_dim]  token stride out_tok_stride
 * max_seqlen_q / max_seqlen_k bound the segment lengths (as in FA2; they size
 * the launch grid).  A caller that understates them gets what FA2 gives:
 * a segment longer than max_seqlen_q has rows the grid does not cover, left
 * unwritten (here the segment's first rows, since causal q-blocks are
 * numbered from its end), and only its first max_seqlen_k keys are
 * attended; no access leaves the segment's rows.  Built for dtype
 * BF16/FP16, head_dim 128, group 1/2/4/8.  With too few work items for the
 * GPU -- one or a few long requests -- the keys of each item are split over its
 * workgroup's waves (groups 2, 4 and 8) or over two workgroups whose partial
 * results are merged by a log-sum-exp combine (in a fixed order: results are the
 * same on every run).  The latter, group 1's and that of groups with many more
 * keys than queries, needs `workspace` of
 * aac_prefill_workspace_bytes(...) bytes, 256-byte aligned, ZERO-FILLED
 * ONCE when it is allocated: its first 16 KiB are per-item counters that
 * every call leaves at zero again, the rest partial results (do not share
 * it with other data or with calls that overlap on another stream).
 * workspace NULL, too small or misaligned: the call runs without a split.
 * Replaces flash_attn_varlen_func (llm.py:178-184).
 */
int aac_prefill_varlen(const void* q, const void* k, const void* v, int64_t q_tok_stride,
                       int64_t k_tok_stride, int64_t v_tok_stride, const int32_t* cu_seqlens_q,
                       const int32_t* cu_seqlens_k, int32_t n_seqs, int32_t max_seqlen_q,
                       int32_t max_seqlen_k, int32_t n_q_heads, int32_t n_kv_heads,
                       int32_t head_dim, float scale, int32_t causal, void* out,
                       int64_t out_tok_stride, void* workspace, size_t workspace_bytes,
                       int32_t dtype, void* stream);

/*
 * Workspace bytes aac_prefill_varlen would use to split this shape's key
 * ranges over two workgroups on the current device (0: it would not).
 */
size_t aac_prefill_workspace_bytes(int32_t n_seqs, int32_t max_seqlen_q, int32_t max_seqlen_k,
                                   int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                   int32_t causal);

/*
 * The result of aac_kv_store(k, v -> caches via slot_mapping) followed by
 * aac_prefill_varlen on the same stream: the whole per-layer attention block
 * of the reference's prefill (llm.py:171-184).  slot_mapping has n_kv_tokens
 * entries, one per packed key token (n_kv_tokens = cu_seqlens_k[n_seqs]);
 * every one of them is stored, also tokens outside all segments.  Causal
 * self-attention (cu_seqlens_q == cu_seqlens_k as pointers, equal max_seqlen)
 * runs as one kernel that stores each q-block's K/V rows after attending to
 * them; other calls launch the store, then the attention.  This call never
 * splits key ranges (no workspace).
 */
int aac_prefill_varlen_store(const void* q, const void* k, const void* v, int64_t q_tok_stride,
                             int64_t k_tok_stride, int64_t v_tok_stride,
                             const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                             int32_t n_seqs, int32_t max_seqlen_q, int32_t max_seqlen_k,
                             int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, float scale,
                             int32_t causal, void* out, int64_t out_tok_stride, void* k_cache,
                             void* v_cache, int64_t num_cache_rows, const int64_t* slot_mapping,
                             int64_t n_kv_tokens, int32_t dtype, void* stream);

/*
 * Bytes of split-K workspace aac_decode_paged needs for this shape.
 * max_context_len <= 0 means "table capacity" (max_blocks_per_seq *
 * block_size), partition_tokens <= 0 means "library's choice".  Returns 0
 * when the chosen plan needs no workspace.
 */
size_t aac_decode_workspace_bytes(int32_t n_seqs, int32_t n_q_heads, int32_t n_kv_heads,
                                  int32_t head_dim, int32_t block_size, int32_t max_blocks_per_seq,
                                  int32_t max_context_len, int32_t partition_tokens);

/*
 * Paged decode attention: one query token per sequence,
 *   out[b, h] = softmax(scale * q[b, h] . K_b^T) V_b
 * over the first context_lens[b] tokens of sequence b, located through
 * block_tables[b * max_blocks_per_seq + i] (physical block of tokens
 * [i*block_size, (i+1)*block_size)).  context_lens[b] == 0 gives zeros; a
 * context longer than the table capacity is clamped to it.  Block ids outside
 * [0, num_blocks) are read as block 0 (output undefined, memory safe).
 *   q   [n_seqs, n_q_heads, head_dim]  seq stride q_seq_stride
 *   out [n_seqs, n_q_heads, head_dim]  seq stride out_seq_stride
 * Long contexts are split into partitions of partition_tokens (<= 0: auto)
 * that are combined with a log-sum-exp reduction in `workspace`
 * (aac_decode_workspace_bytes).  max_context_len (<= 0: table capacity) is
 * an upper bound on context_lens used to size the grid.
 * Built for dtype BF16/FP16/FP32, head_dim 128, group 1/2/4/8.
 * Replaces the attend half of flash_attn_with_kvcache (model/model.py:233-240).
 */
int aac_decode_paged(const void* q, int64_t q_seq_stride, const void* k_cache, const void* v_cache,
                     int64_t num_blocks, int32_t block_size, const int32_t* block_tables,
                     int32_t max_blocks_per_seq, const int32_t* context_lens, int32_t n_seqs,
                     int32_t max_context_len, int32_t n_q_heads, int32_t n_kv_heads,
                     int32_t head_dim, float scale, void* out, int64_t out_seq_stride,
                     void* workspace, size_t workspace_bytes, int32_t partition_tokens,
                     int32_t dtype, void* stream);

/* Bytes of the static split-K scratch aac_decode_paged_noalloc uses. */
#define AAC_DECODE_SCRATCH_BYTES (64u << 20)

/*
 * aac_decode_paged without a workspace: the same kernels, plan and results,
 * with the split-K partials in a static device array of
 * AAC_DECODE_SCRATCH_BYTES that the library holds on each GPU it runs on
 * until the process ends.  Allocates nothing (no hipMalloc, no library
 * allocation): for callers that cannot allocate device memory -- code under
 * HIP graph capture, tight serving loops, harnesses that forbid it.  A plan
 * whose workspace (aac_decode_workspace_bytes) exceeds the scratch returns
 * AAC_ERR_SCRATCH before anything is enqueued.  Every call on a GPU shares
 * that GPU's array (the device current on the calling thread), so calls
 * that overlap on one GPU -- other streams or threads -- race and must be
 * serialised by the caller; each call writes every scratch slot it reads, so
 * nothing carries over between calls.
 * No counterpart in the reference: an extra for callers that cannot
 * allocate.
 */
int aac_decode_paged_noalloc(const void* q, int64_t q_seq_stride, const void* k_cache,
                             const void* v_cache, int64_t num_blocks, int32_t block_size,
                             const int32_t* block_tables, int32_t max_blocks_per_seq,
                             const int32_t* context_lens, int32_t n_seqs,
                             int32_t max_context_len, int32_t n_q_heads, int32_t n_kv_heads,
                             int32_t head_dim, float scale, void* out, int64_t out_seq_stride,
                             int32_t partition_tokens, int32_t dtype, void* stream);

/*
 * flash_attn_with_kvcache(q, k_cache, v_cache, k=k, v=v, cache_seqlens,
 * block_table, softmax_scale, causal=False): append k/v at position
 * cache_seqlens[b] (aac_kv_append_paged), then attend over
 * cache_seqlens[b] + 1 tokens.  cache_seqlens is not modified.
 * max_context_len bounds cache_seqlens[b] + 1 (<= 0: table capacity).
 * The append runs inside the attention launch with the result of an append
 * before it: every row of the call sees the new tokens of all rows in blocks that
 * its table shares with them (one sequence given as several rows, at positions n,
 * n + 1, ...).  Two rows that write the same cache row: one of them stays in the
 * cache.
 * Replaces model/model.py:233-240.
 */
int aac_decode_append_paged(const void* q, int64_t q_seq_stride, const void* k, const void* v,
                            int64_t k_tok_stride, int64_t v_tok_stride, void* k_cache,
                            void* v_cache, int64_t num_blocks, int32_t block_size,
                            const int32_t* block_tables, int32_t max_blocks_per_seq,
                            const int32_t* cache_seqlens, int32_t n_seqs, int32_t max_context_len,
                            int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, float scale,
                            void* out, int64_t out_seq_stride, void* workspace,
                            size_t workspace_bytes, int32_t partition_tokens, int32_t dtype,
                            void* stream);

/*
 * aac_decode_append_paged with counters (8 bytes per (sequence, KV head), 8-byte
 * aligned, or null): a small split call then combines its partitions in the
 * attention launch instead of a second one.  One launch less for a caller that
 * launches each call itself; slower on the GPU from some 4 partitions on, so a
 * captured step passes null.  The counters need no initialisation; like the
 * workspace they belong to one call at a time.
 */
int aac_decode_append_merge_paged(
    const void* q, int64_t q_seq_stride, const void* k, const void* v, int64_t k_tok_stride,
    int64_t v_tok_stride, void* k_cache, void* v_cache, int64_t num_blocks, int32_t block_size,
    const int32_t* block_tables, int32_t max_blocks_per_seq, const int32_t* cache_seqlens,
    int32_t n_seqs, int32_t max_context_len, int32_t n_q_heads, int32_t n_kv_heads,
    int32_t head_dim, float scale, void* out, int64_t out_seq_stride, void* workspace,
    size_t workspace_bytes, void* counters, int32_t partition_tokens, int32_t dtype, void* stream);

/*
 * The same step from the rows of the fused QKV projection, qkv
 * [n_seqs, (n_q_heads + 2 n_kv_heads) * head_dim]: q/k RMSNorm + RoPE at
 * positions[b] (model/model.py:219-228, as aac_qk_norm_rope_store), the append
 * of k and v at cache_seqlens[b], and the attention over cache_seqlens[b] + 1
 * tokens (model/model.py:233-240), without the normalised q and k in memory.
 * Rows that share blocks see each other's new tokens, as above.
 * dtype bf16 or fp16; the workspace is aac_decode_workspace_bytes'.
 */
int aac_decode_qkv_paged(const void* qkv, int64_t qkv_row_stride, const void* q_norm_weight,
                         const void* k_norm_weight, float eps, const void* cos_table,
                         const void* sin_table, int32_t max_position, const int32_t* positions,
                         void* k_cache, void* v_cache, int64_t num_blocks, int32_t block_size,
                         const int32_t* block_tables, int32_t max_blocks_per_seq,
                         const int32_t* cache_seqlens, int32_t n_seqs, int32_t max_context_len,
                         int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, float scale,
                         void* out, int64_t out_seq_stride, void* workspace,
                         size_t workspace_bytes, int32_t partition_tokens, int32_t dtype,
                         void* stream);

/* ------------------------------------------------------------------------
 * Fused kernels of the attention call site.  Each replaces a chain of small
 * torch kernels of the reference layer with one launch and rounds to the
 * activation dtype at the same points.  dtype: BF16 or FP16.
 * ---------------------------------------------------------------------- */

/*
 * out = weight * dtype(h * rsqrt(mean(h^2) + eps)), statistics in fp32, where
 * h = x, or h = dtype(x + residual) with residual_out = h when residual is
 * given (residual and residual_out together or neither).  x rows have stride
 * x_row_stride; residual, residual_out and out are contiguous [n_rows, hidden].
 * hidden must be a multiple of 512, at most 4096.
 * Replaces RMSNorm (model/model.py:47-52) and the residual add before it
 * (model/model.py:259, :265; llm.py:188, :194).
 */
int aac_rmsnorm(const void* x, int64_t x_row_stride, const void* residual, void* residual_out,
                const void* weight, void* out, int64_t n_rows, int32_t hidden, float eps,
                int32_t dtype, void* stream);

/*
 * Per token of the fused QKV projection qkv [n_tokens, (Hq + 2*Hkv) * 128]
 * (row stride qkv_tok_stride): RMSNorm of every q and k head with
 * q_norm_weight / k_norm_weight, then RoPE with the cos/sin tables
 * [max_position, 128] at positions[t] (x*cos + rotate_half(x)*sin, each term
 * rounded), writing q_out [n_tokens, Hq, 128] and, if k_out is given,
 * k_out [n_tokens, Hkv, 128].  If v_cache is given the rotated k and the raw v
 * of token t are stored in the caches (rows [*, Hkv, 128]): at row
 * slot_mapping[t] (negative or >= num_cache_rows: skipped), or, when
 * slot_mapping is NULL, appended at position cache_seqlens[t] of block table
 * row t (decode: token t is sequence t).
 * Replaces model/model.py:219-228 plus the KV store llm.py:171-174 /
 * the k=/v= append of flash_attn_with_kvcache (model/model.py:233-240).
 */
int aac_qk_norm_rope_store(const void* qkv, int64_t qkv_tok_stride, int64_t n_tokens,
                           int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                           const void* q_norm_weight, const void* k_norm_weight, float eps,
                           const void* cos_table, const void* sin_table, int32_t max_position,
                           const int32_t* positions, void* q_out, void* k_out, void* k_cache,
                           void* v_cache, int64_t num_cache_rows, const int64_t* slot_mapping,
                           const int32_t* block_tables, int32_t max_blocks_per_seq,
                           const int32_t* cache_seqlens, int32_t block_size, int32_t dtype,
                           void* stream);

/*
 * out[r, i] = dtype(silu(gate_up[r, i])) * gate_up[r, intermediate + i] for the
 * fused [gate | up] projection gate_up [n_rows, 2*intermediate].
 * Replaces act_fn(gate_proj(x)) * up_proj(x) (model/model.py:188).
 */
int aac_silu_mul(const void* gate_up, void* out, int64_t n_rows, int32_t intermediate,
                 int32_t dtype, void* stream);

/*
 * Decode-batch projection: y[m, n] = sum_k x[m, k] * w[n, k] (torch's
 * F.linear(x, w), fp32 accumulation, rounded to dtype) for x [m, k] and a
 * Linear weight w [n, k], rows strided by *_row_stride elements.  With
 * silu_intermediate = I (> 0) the weight is the fused [gate | up] projection
 * [2I, k], n must equal I, and y[m, i] = dtype(silu(dtype(gate))) *
 * dtype(up), the rounding of act_fn(gate_proj(x)) * up_proj(x)
 * (model/model.py:188) -- the product of aac_silu_mul without the [m, 2I]
 * intermediate.  Built for shapes where n is a multiple of 32 and k of 64
 * (of 128 / 256 for some tilings); config 0 lets the library pick the tiling,
 * 1..6 force one (tuning; a tiling whose stages do not fit LDS with the
 * gate/up pairing returns AAC_ERR_UNSUPPORTED).  Meant for the small m of a decode step (tens to
 * hundreds of rows): every output tile is one workgroup.
 * Replaces the q/k/v, o_proj, gate/up and down nn.Linear calls of the
 * decoder layer (model/model.py:132-154, :258, :178-188) on decode steps.
 */
int aac_gemm_nt(const void* x, int64_t x_row_stride, const void* w, int64_t w_row_stride, void* y,
                int64_t y_row_stride, int32_t m, int32_t n, int32_t k, int32_t silu_intermediate,
                int32_t config, int32_t dtype, void* stream);

/*
 * The fused QKV projection of a decode step followed by aac_qk_norm_rope_store
 * in one launch: qkv = x w_qkv^T (x [n_tokens, hidden], w_qkv the fused
 * [(Hq + 2*Hkv) * 128, hidden] weight, fp32 accumulation rounded to dtype
 * exactly as aac_gemm_nt's tiling 6 rounds it), then per token the q/k
 * RMSNorm + RoPE of every q and k head and the K/V store or decode append,
 * with the arguments and results of aac_qk_norm_rope_store (the [n_tokens,
 * Hq+2Hkv, 128] qkv intermediate is never written).  hidden must be a
 * multiple of 128.  Replaces the QKV projection and model/model.py:219-228
 * plus the k=/v= append of flash_attn_with_kvcache (model/model.py:233-240).
 */
int aac_qkv_norm_rope_store(const void* x, int64_t x_row_stride, const void* w_qkv,
                            int64_t w_row_stride, int64_t n_tokens, int32_t hidden,
                            int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                            const void* q_norm_weight, const void* k_norm_weight, float eps,
                            const void* cos_table, const void* sin_table, int32_t max_position,
                            const int32_t* positions, void* q_out, void* k_out, void* k_cache,
                            void* v_cache, int64_t num_cache_rows, const int64_t* slot_mapping,
                            const int32_t* block_tables, int32_t max_blocks_per_seq,
                            const int32_t* cache_seqlens, int32_t block_size, int32_t dtype,
                            void* stream);

/*
 * aac_gemm_nt with the residual add and RMSNorm of aac_rmsnorm in its
 * prologue, for a decode step of few rows: h = x, or h = dtype(x + residual)
 * with residual_out = h when residual is given (both contiguous [m, k]),
 * y = norm(h) w^T (with silu_intermediate: SiLU * up).  k is 512 or 1024 and n a
 * multiple of 32, else AAC_ERR_UNSUPPORTED.  Not in place: residual_out and y share
 * no byte with x, residual or each other, else AAC_ERR_INVALID_ARGUMENT.
 */
int aac_rmsnorm_gemm_nt(const void* x, int64_t x_row_stride, const void* residual,
                        void* residual_out, const void* norm_weight, float eps, const void* w,
                        int64_t w_row_stride, void* y, int64_t y_row_stride, int32_t m, int32_t n,
                        int32_t k, int32_t silu_intermediate, int32_t dtype, void* stream);

/*
 * Greedy sampling: out[r] = the index of the largest element of row r of x
 * [n_rows, n_cols] (row stride row_stride elements; BF16, FP16 or FP32), the
 * first one among equal maxima, a NaN counting as the largest -- the result
 * of torch.argmax(dim=-1).  Replaces logits.argmax(dim=-1) of the sampler
 * (llm.py:215-219, temperature 0).
 */
int aac_argmax_rows(const void* x, int64_t row_stride, int64_t n_rows, int64_t n_cols,
                    int64_t* out, int32_t dtype, void* stream);

/*
 * KV export: gather the first `length` tokens of one sequence from a paged
 * cache into a contiguous buffer out[n_layers][2][length][Hkv][D] (index 0 =
 * K, 1 = V).  Layer l's K cache starts at kv_cache + l * layer_stride and its
 * V cache kv_stride elements after that (both [num_blocks, block_size, Hkv,
 * D]); token t lives in block block_table[t / block_size] (table width
 * max_blocks; length <= max_blocks * block_size).  Entries outside
 * [0, num_blocks) export zeros.  Replaces the per-layer slices
 * k_cache[slot, :length] / v_cache[slot, :length] of export_kv and
 * export_request_kv (model/model.py:156-165, :386-390); the slot layout is
 * block_table = [slot], block_size = max_seq_len.
 */
int aac_kv_export_paged(const void* kv_cache, int64_t layer_stride, int64_t kv_stride,
                        int32_t n_layers, int64_t num_blocks, int32_t block_size,
                        int32_t n_kv_heads, int32_t head_dim, const int32_t* block_table,
                        int32_t max_blocks, int32_t length, void* out, int32_t dtype,
                        void* stream);

/*
 * KV import: scatter src[n_layers][2][length][Hkv][D] into the paged cache
 * through block_table (same layout and arguments as aac_kv_export_paged);
 * entries outside [0, num_blocks) are skipped.  Replaces the per-layer
 * copy_ of import_kv and import_request_kv (model/model.py:167-177, :392-401);
 * cache_seqlens stays with the caller, as the reference sets it separately.
 */
int aac_kv_import_paged(const void* src, void* kv_cache, int64_t layer_stride, int64_t kv_stride,
                        int32_t n_layers, int64_t num_blocks, int32_t block_size,
                        int32_t n_kv_heads, int32_t head_dim, const int32_t* block_table,
                        int32_t max_blocks, int32_t length, int32_t dtype, void* stream);

/*
 * The paged KV cache in four bits.  cache: uint8 [num_blocks][n_kv_heads][K, V]
 * [block_size * 68], 64-byte aligned, block_size a multiple of 16 (to 2^23), head_dim 128.  A
 * page holds block_size rows of 64 bytes (E2M1 codes, dim 2 i in the low nibble of
 * byte i), then block_size rows of 4 scale bytes (E8M0, one for 32 dims): an element
 * is code * 2^(byte - 127), NaN where the byte is 255.  With a = max |x| of 32 dims, the
 * store sets byte - 127 = (exponent of a rounded to two significant bits) - 2, within
 * [-125, 125], and rounds x / 2^(byte - 127) to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6,
 * halves to the even code; 32 dims with an infinity or a NaN are stored as NaN.
 *
 * aac_kv4_store: row slot_mapping[t] of the cache (block slot / block_size, row slot
 * mod block_size) gets k[t] and v[t]; slots outside the cache (negative: padding) are
 * skipped.  Slots are distinct: a row named twice holds parts of both.
 * aac_kv4_append: the same for one token a sequence at position cache_seqlens[b], as
 * aac_kv_append_paged.
 * aac_kv4_load: k_out[t], v_out[t] ([n_tokens, n_kv_heads, 128], 16-byte aligned) =
 * the values of row slot_mapping[t], rounded to dtype; zeros for a slot outside.
 * dtype BF16, FP16 or FP32; k and v have any token stride and alignment.
 */
int aac_kv4_store(const void* k, const void* v, int64_t k_tok_stride, int64_t v_tok_stride,
                  void* cache, int64_t num_blocks, int32_t block_size, const int64_t* slot_mapping,
                  int64_t n_tokens, int32_t n_kv_heads, int32_t head_dim, int32_t dtype,
                  void* stream);
int aac_kv4_append(const void* k, const void* v, int64_t k_seq_stride, int64_t v_seq_stride,
                   void* cache, int64_t num_blocks, int32_t block_size, const int32_t* block_tables,
                   int32_t max_blocks_per_seq, const int32_t* cache_seqlens, int32_t n_seqs,
                   int32_t n_kv_heads, int32_t head_dim, int32_t dtype, void* stream);
int aac_kv4_load(const void* cache, int64_t num_blocks, int32_t block_size,
                 const int64_t* slot_mapping, int64_t n_tokens, int32_t n_kv_heads, int32_t head_dim,
                 void* k_out, void* v_out, int32_t dtype, void* stream);

/*
 * aac_qk_norm_rope_store with the 4-bit cache in the place of the 16-bit caches: q/k
 * RMSNorm + RoPE of the fused projection, and k (rounded to dtype) and v quantised into
 * the rows slot_mapping names or, where it is null, appended at cache_seqlens of
 * block_tables.  q_out [n_tokens, n_q_heads, 128]; k_out [n_tokens, n_kv_heads, 128] or
 * null.  The cache holds what aac_kv4_store of k_out and v would write.  BF16 or FP16.
 */
int aac_qk_norm_rope_store_kv4(
    const void* qkv, int64_t qkv_tok_stride, int64_t n_tokens, int32_t n_q_heads, int32_t n_kv_heads,
    int32_t head_dim, const void* q_norm_weight, const void* k_norm_weight, float eps,
    const void* cos_table, const void* sin_table, int32_t max_position, const int32_t* positions,
    void* q_out, void* k_out, void* cache, int64_t num_blocks, int32_t block_size,
    const int64_t* slot_mapping, const int32_t* block_tables, int32_t max_blocks_per_seq,
    const int32_t* cache_seqlens, int32_t dtype, void* stream);

/*
 * Decode over the 4-bit cache: out[b] = softmax(scale q[b] K^T) V over the first
 * context_lens[b] tokens of sequence b (at most the table's capacity and 2^31 - 1024;
 * none: zeros), read through block_tables as aac_decode_paged reads them.  With k and v (one row of
 * n_kv_heads * 128 a sequence, dtype as q's) they are appended first, at position
 * context_lens[b], as aac_kv4_append does, and the call attends over one token more; all
 * rows are written before any is read.  Both null: attend only.
 * q, out [n_seqs, n_q_heads, 128] BF16, FP16 or FP32; n_q_heads / n_kv_heads from 1 to 16.
 * max_context_len: 0, or a bound on every context (what lies past it may be left out).
 * Contexts split over workgroups need aac_kv4_decode_workspace_bytes(...) bytes of
 * workspace, 16-byte aligned, any contents, not shared with a call that may overlap.
 * partition_tokens: 0, or the tokens of a partition (rounded up to 256).
 */
size_t aac_kv4_decode_workspace_bytes(int32_t n_seqs, int32_t n_q_heads, int32_t n_kv_heads,
                                      int32_t head_dim, int32_t block_size,
                                      int32_t max_blocks_per_seq, int32_t max_context_len,
                                      int32_t partition_tokens);
int aac_kv4_decode(const void* q, int64_t q_seq_stride, const void* k, const void* v,
                   int64_t k_seq_stride, int64_t v_seq_stride, void* cache, int64_t num_blocks,
                   int32_t block_size, const int32_t* block_tables, int32_t max_blocks_per_seq,
                   const int32_t* context_lens, int32_t n_seqs, int32_t max_context_len,
                   int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                   float scale, void* out, int64_t out_seq_stride, void* workspace,
                   size_t workspace_bytes, int32_t partition_tokens, int32_t dtype, void* stream);

/*
 * A step's maps from its request lengths.  Sequence b holds cached_lens[b] tokens (null:
 * none) and gets new_lens[b] more (negative lengths count as 0; the new ones sum to less
 * than 2^31):
 *   cu_seqlens [n_seqs + 1]  prefix sums of new_lens
 *   positions, slot_mapping [n_tokens]  of token i of sequence b, at cu_seqlens[b] + i:
 *       cached_lens[b] + i, and its cache row through the block table; a slot is -1
 *       without a block or past the table, and behind the last sequence (position 0)
 *   context_lens [n_seqs]  cached + new
 * With free_blocks (n_free of them) the blocks a sequence needs beyond the
 * ceil(cached / block_size) it holds are taken from it in order, sequence by sequence,
 * and written to block_tables; past its end they are -1.  blocks_taken[0] = the blocks
 * asked for: more than n_free means that some are missing.  Null: the tables are
 * complete and only read.  n_seqs up to AAC_STEP_MAPS_MAX_SEQS.
 * Replaces the host's metadata construction (llm.py:127-140).
 */
#define AAC_STEP_MAPS_MAX_SEQS 8192
int aac_step_maps(const int32_t* new_lens, const int32_t* cached_lens, int32_t* block_tables,
                  int32_t n_seqs, int32_t max_blocks_per_seq, int32_t block_size,
                  const int32_t* free_blocks, int32_t n_free, int64_t n_tokens,
                  int32_t* cu_seqlens, int64_t* positions, int64_t* slot_mapping,
                  int32_t* context_lens, int32_t* blocks_taken, void* stream);

/*
 * For each row of logits [n_rows, n_cols] (row stride row_stride elements, any
 * alignment; BF16, FP16 or FP32): logprobs[r] = log softmax(row)[tokens[r]] (0 for a
 * negative token, NaN for one past the row), entropy[r] of the softmax, and the top_k
 * (0 to AAC_LOGPROBS_MAX_TOP, at most n_cols) largest: top_logprobs, top_ids [n_rows,
 * top_k], the first index first among equal logits, a NaN counting as the largest.  A
 * row with a NaN or +inf, or of -inf alone, gets NaN, as torch.log_softmax.
 * n_cols up to AAC_LOGPROBS_MAX_COLS.  workspace: aac_logprobs_workspace_bytes(...) bytes,
 * 16-byte aligned, any contents, not shared with a call that may overlap.
 */
#define AAC_LOGPROBS_MAX_TOP 32
#define AAC_LOGPROBS_MAX_COLS (1 << 20)
size_t aac_logprobs_workspace_bytes(int64_t n_rows, int64_t n_cols, int32_t top_k);
int aac_token_logprobs(const void* logits, int64_t row_stride, int64_t n_rows, int64_t n_cols,
                       const int64_t* tokens, int32_t top_k, float* logprobs, float* entropy,
                       float* top_logprobs, int64_t* top_ids, void* workspace,
                       size_t workspace_bytes, int32_t dtype, void* stream);

/*
 * Attention of a chunk of new tokens over the paged cache.  Sequence b's queries are rows
 * [cu_seqlens_q[b], cu_seqlens_q[b+1]) of q [n_tokens, n_q_heads, head_dim] (token stride
 * q_tok_stride), or, where cu_seqlens_q is null, max_seqlen_q rows each; its keys are the
 * first L_b tokens of its blocks, L_b = context_lens[b] or, where that is null,
 * cu_seqlens_k[b+1] - cu_seqlens_k[b] (the new tokens' rows among them: they are stored first).  With causal != 0 the mask is bottom-right aligned: query i
 * of n sees keys j <= i + L_b - n.  A query that sees no key gets zeros; what a masked key's
 * value or a row behind the context holds, infinities and NaN too, reaches no query that
 * does not see it.  Rows of q behind the last sequence are left as they are in out.
 * Tables as in aac_decode_paged: a context longer than the table is cut to it, block ids
 * outside [0, num_blocks) are read as block 0.  max_seqlen_q: an upper bound on the
 * sequences' queries (of a longer one, rows past it may be left unwritten);
 * max_context_len (<= 0: the table's capacity): an estimate of the longest context, which
 * only chooses how the work is split.
 * BF16 or FP16, head_dim 128, n_q_heads any multiple (below 2^14) of n_kv_heads, scale > 0.  A
 * table of more than one block whose size is not a multiple of 16 names 2^27 tokens at most.
 * workspace: aac_prefill_paged_workspace_bytes(...) bytes (the same arguments) where
 * that is not 0, 16-byte aligned, any contents, not shared with a call that may overlap.
 */
size_t aac_prefill_paged_workspace_bytes(int64_t n_tokens, int32_t n_seqs, int32_t max_seqlen_q,
                                         int32_t max_context_len, int32_t block_size,
                                         int32_t max_blocks_per_seq, int32_t n_q_heads,
                                         int32_t n_kv_heads);
int aac_prefill_paged(const void* q, int64_t q_tok_stride, int64_t n_tokens, const void* k_cache,
                      const void* v_cache, int64_t num_blocks, int32_t block_size,
                      const int32_t* block_tables, int32_t max_blocks_per_seq,
                      const int32_t* cu_seqlens_q, const int32_t* context_lens,
                      const int32_t* cu_seqlens_k, int32_t n_seqs, int32_t max_seqlen_q,
                      int32_t max_context_len, int32_t n_q_heads, int32_t n_kv_heads,
                      int32_t head_dim, float scale, int32_t causal, void* out,
                      int64_t out_tok_stride, void* workspace, size_t workspace_bytes,
                      int32_t dtype, void* stream);

/*
 * Rotary positions.  The first rotary_dim dims of a head are rotary_dim / 2 pairs, (d, d +
 * rotary_dim / 2) or, interleaved, (2 d, 2 d + 1); pair d of a token at position p becomes
 * (x1 c - x2 s, x1 s + x2 c) with c, s = cos_table, sin_table [table_rows, rotary_dim / 2]
 * at (p, d): in fp32, rounded once.  The other dims pass unchanged.  Positions outside the
 * tables take their first or last row.  dtype BF16, FP16 or FP32; table_dtype dtype or
 * FP32; head_dim even, rotary_dim even and at most head_dim.  Head strides are free.
 * A call takes a wave for every 4 KiB of a token's rows that it turns or stores, begun or whole;
 * 2^26 waves and more are refused.
 *
 * aac_rotary: x -> out (out may be x).  Without cu_seqlens: [n_seqs, seqlen, n_heads,
 * head_dim] by its strides, token i of sequence b at position offsets[b] + i (offsets null:
 * offset + i); n_tokens is not read.  With cu_seqlens [n_seqs + 1]: packed [n_tokens,
 * n_heads, head_dim] (the sequence strides are not read), token cu_seqlens[b] + i at
 * position offsets[b] + i; rows of no sequence are left as they are.  conjugate != 0 turns
 * back.
 *
 * aac_rotary_append_paged: new token i of sequence b, at position cache_seqlens[b] + i: its
 * key turned and its value as it is into the row its block table names for that position
 * (none: skipped, as aac_kv_append_paged), its queries turned into q_out (contiguous, as q
 * is shaped; q null: no queries).  Without cu_seqlens q is [n_seqs, seqlen_q, ...] and k,
 * v [n_seqs, seqlen_k, ...]; with it all are packed [n_tokens, ...].  queries_at_first !=
 * 0: every query of a sequence turns at cache_seqlens[b].  rotary_dim 0: the append alone
 * (q is copied).  cache_seqlens is not modified; context_lens (or null; without
 * cu_seqlens) gets cache_seqlens[b] + seqlen_k.
 * The k= / v= / rotary_cos= half of flash_attn_with_kvcache (model/model.py:233-240).
 *
 * aac_rotary_tables: cos_out, sin_out [n_positions, n_freqs] = factor * cos, sin of
 * 2 pi p turns[i] at positions p = positions[r] or, where that is null, start + r.  turns:
 * double [n_freqs] on the device, turns a position, 1 at most; the angle is reduced in 64
 * bits.  |start| up to 2^40, fewer than 2^32 vectors of 16 bytes in an output; cos_out and sin_out 16-byte aligned where n_freqs is a multiple of 8 (FP32: of 4).
 */
int aac_rotary(const void* x, int64_t x_seq_stride, int64_t x_tok_stride, int64_t x_head_stride,
               void* out, int64_t out_seq_stride, int64_t out_tok_stride, int64_t out_head_stride,
               int32_t n_seqs, int32_t seqlen, int64_t n_tokens, const int32_t* cu_seqlens,
               const int32_t* offsets, int32_t offset, int32_t n_heads, int32_t head_dim,
               const void* cos_table, const void* sin_table, int32_t table_rows,
               int32_t rotary_dim, int32_t interleaved, int32_t conjugate, int32_t table_dtype,
               int32_t dtype, void* stream);
int aac_rotary_append_paged(
    const void* q, int64_t q_seq_stride, int64_t q_tok_stride, int64_t q_head_stride, const void* k,
    int64_t k_seq_stride, int64_t k_tok_stride, int64_t k_head_stride, const void* v,
    int64_t v_seq_stride, int64_t v_tok_stride, int64_t v_head_stride, void* q_out, int32_t n_seqs,
    int32_t seqlen_q, int32_t seqlen_k, int64_t n_tokens, const int32_t* cu_seqlens,
    const int32_t* cache_seqlens, int32_t* context_lens, int32_t n_q_heads, int32_t n_kv_heads,
    int32_t head_dim, const void* cos_table, const void* sin_table, int32_t table_rows,
    int32_t rotary_dim, int32_t interleaved, int32_t queries_at_first, void* k_cache, void* v_cache, int64_t num_blocks,
    int32_t block_size, const int32_t* block_tables, int32_t max_blocks_per_seq, int32_t table_dtype,
    int32_t dtype, void* stream);
int aac_rotary_tables(const void* turns, int32_t n_freqs, const int32_t* positions, int64_t start,
                      int64_t n_positions, float factor, void* cos_out, void* sin_out, int32_t dtype,
                      void* stream);

#ifdef __cplusplus
}
#endif

#endif /* AAC_ATTN_H */
