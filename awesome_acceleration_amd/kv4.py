"""The paged KV cache in four bits: store, append, load and decode attention.

A cached element is an E2M1 code times a power of two shared by 32 dims (OCP
microscaling FP4), 136 bytes a token and KV head for K and V against 512 in bf16.
The cache is one uint8 tensor ``[num_blocks, Hkv, 2, block_size * 68]``: for each block
and KV head the K page, then the V page; a page holds ``block_size`` rows of 64 bytes
(dim ``2 i`` in the low nibble of byte ``i``) and then ``block_size`` rows of 4 scale
bytes (``2^(byte - 127)``; 255: NaN).  Blocks, block tables and slot mappings are those
of the 16-bit paged cache; ``block_size`` is a multiple of 16 and ``head_dim`` 128.

``kv4_store`` and ``kv4_load`` stand beside ``kv_store`` and the KV export,
``decode_paged_kv4`` and ``flash_attn_with_kv4cache`` beside ``decode_paged`` and
``flash_attn_with_kvcache``, with their conventions: ``RuntimeError`` for a rejected
argument, the current stream, no synchronisation, new outputs, caches updated in place.
Lengths are int32 throughout.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch

from . import _lib
from .flash_attn_interface import (_check_slots, _on_gpu, _require, _scale, _token_rows,
                                   check_mode)

__all__ = ["alloc_kv4_cache", "kv4_store", "kv4_load", "decode_paged_kv4",
           "flash_attn_with_kv4cache", "qk_norm_rope_store_kv4", "kv4_export", "kv4_import",
           "BYTES_PER_TOKEN"]

HEAD_DIM = 128
PAGE_BYTES = 68        # of a token's K or V row of one head: 64 of codes, 4 of scales
BYTES_PER_TOKEN = 136  # K and V of one token and KV head
TILE = 16              # block sizes are multiples of it


def alloc_kv4_cache(num_blocks: int, block_size: int, n_kv_heads: int, head_dim: int = HEAD_DIM, *,
                    device, n_layers: Optional[int] = None) -> torch.Tensor:
    """A zero-filled cache (every value 0), ``[num_blocks, Hkv, 2, block_size * 68]``,
    with ``n_layers`` in front where given."""
    _require(head_dim == HEAD_DIM, f"the 4-bit cache is built for head_dim {HEAD_DIM}")
    _require(block_size > 0 and block_size % TILE == 0, f"block_size must be a multiple of {TILE}")
    shape = (num_blocks, n_kv_heads, 2, block_size * PAGE_BYTES)
    return torch.zeros(shape if n_layers is None else (n_layers, *shape), dtype=torch.uint8,
                       device=device)


def _cache(kv_cache: torch.Tensor) -> tuple[int, int, int]:
    """(num_blocks, block_size, Hkv) of a cache, checked."""
    shape = kv_cache.shape
    if (kv_cache.dtype is not torch.uint8 or len(shape) != 4 or shape[2] != 2
            or not kv_cache.is_contiguous()):
        raise RuntimeError("kv_cache must be contiguous uint8 [num_blocks, Hkv, 2, block_size * 68]")
    bs = shape[3] // PAGE_BYTES
    if shape[3] != bs * PAGE_BYTES or bs == 0 or bs % TILE:
        raise RuntimeError(f"kv_cache pages must be block_size * {PAGE_BYTES} bytes, block_size a "
                           f"multiple of {TILE}")
    return shape[0], bs, shape[1]


def _slots(slot_mapping: torch.Tensor, n: Optional[int]) -> None:
    if (slot_mapping.dtype is not torch.int64 or slot_mapping.dim() != 1
            or not slot_mapping.is_contiguous() or (n is not None and slot_mapping.shape[0] != n)):
        raise RuntimeError("slot_mapping must be contiguous int64 [N]")


def _code(dtype: torch.dtype) -> int:
    code = _lib.AAC_DTYPE.get(dtype)
    if code is None:
        raise RuntimeError(f"unsupported dtype {dtype}")
    return code


def kv4_store(k: torch.Tensor, v: torch.Tensor, kv_cache: torch.Tensor,
              slot_mapping: torch.Tensor) -> None:
    """Quantise ``k``/``v`` (``[N, Hkv, 128]``, any token stride; bf16, fp16 or fp32) into
    the cache rows ``slot_mapping`` (int64 ``[N]``), as ``kv_store`` stores them: negative
    and out-of-range slots are skipped, ``IndexError`` for them with ``AAC_CHECK=1``.
    Slots are distinct (a row named twice holds parts of both tokens)."""
    _on_gpu(k, v, kv_cache, slot_mapping)
    nb, bs, hkv = _cache(kv_cache)
    ks, vs = _token_rows(k, "k"), _token_rows(v, "v")
    shape = k.shape
    if shape != v.shape or k.dtype is not v.dtype:
        raise RuntimeError("k and v must have one shape and dtype")
    if shape[1] != hkv or shape[2] != HEAD_DIM:
        raise RuntimeError("row shape != [Hkv, 128]")
    _slots(slot_mapping, shape[0])
    if check_mode():
        _check_slots(slot_mapping, nb * bs)
    _lib.launch("aac_kv4_store", k.get_device(), k.data_ptr(), v.data_ptr(), ks, vs,
                kv_cache.data_ptr(), nb, bs, slot_mapping.data_ptr(), shape[0], hkv, HEAD_DIM,
                _code(k.dtype))


def kv4_load(kv_cache: torch.Tensor, slot_mapping: torch.Tensor,
             dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The K and V rows ``[N, Hkv, 128]`` that the cache holds at ``slot_mapping`` (int64
    ``[N]``), in ``dtype`` (bf16 and fp32 hold them exactly, fp16 those within its range);
    zeros for a slot outside the cache."""
    _on_gpu(kv_cache, slot_mapping)
    nb, bs, hkv = _cache(kv_cache)
    _slots(slot_mapping, None)
    code = _code(dtype)
    n = slot_mapping.shape[0]
    k = torch.empty((n, hkv, HEAD_DIM), dtype=dtype, device=kv_cache.device)
    v = torch.empty_like(k)
    _lib.launch("aac_kv4_load", kv_cache.get_device(), kv_cache.data_ptr(), nb, bs,
                slot_mapping.data_ptr(), n, hkv, HEAD_DIM, k.data_ptr(), v.data_ptr(), code)
    return k, v


def qk_norm_rope_store_kv4(qkv: torch.Tensor, n_q_heads: int, q_norm_weight: torch.Tensor,
                           k_norm_weight: torch.Tensor, eps: float, cos: torch.Tensor,
                           sin: torch.Tensor, positions: torch.Tensor, kv_cache: torch.Tensor, *,
                           slot_mapping: Optional[torch.Tensor] = None,
                           block_tables: Optional[torch.Tensor] = None,
                           cache_seqlens: Optional[torch.Tensor] = None, want_k: bool = True):
    """``fused.qk_norm_rope_store`` with the 4-bit cache: q/k RMSNorm + RoPE of the fused
    projection ``qkv`` ``[T, (Hq + 2 Hkv) * 128]`` (bf16 or fp16), and the K and V rows
    quantised into the rows of ``slot_mapping`` or appended at ``cache_seqlens`` of
    ``block_tables``, in one launch.  Returns ``(q [T, Hq, 128], k [T, Hkv, 128] or None)``;
    the cache holds what ``kv4_store`` of ``k`` and ``v`` would write."""
    _on_gpu(qkv, q_norm_weight, k_norm_weight, cos, sin, positions, kv_cache, slot_mapping, block_tables,
            cache_seqlens)
    nb, bs, hkv = _cache(kv_cache)
    _require(qkv.dim() == 2 and qkv.stride(1) == 1
             and qkv.shape[1] == (n_q_heads + 2 * hkv) * HEAD_DIM, "qkv must be [T, (Hq + 2 Hkv) * 128]")
    n, dt = qkv.shape[0], qkv.dtype
    _require(dt in (torch.bfloat16, torch.float16), "bf16 and fp16 only")
    for t in (q_norm_weight, k_norm_weight):
        _require(t.dtype is dt and t.shape == (HEAD_DIM,) and t.is_contiguous(), "norm weights must be [128]")
    _require(cos.dim() == 2 and cos.shape[1] == HEAD_DIM and sin.shape == cos.shape and cos.dtype is dt
             and sin.dtype is dt and cos.is_contiguous() and sin.is_contiguous(), "cos/sin must be [P, 128]")
    _require(positions.dtype is torch.int32 and positions.shape == (n,) and positions.is_contiguous(),
             "positions must be contiguous int32 [T]")
    slots = tables = lens = None
    mb = 0
    if slot_mapping is not None:
        _slots(slot_mapping, n)
        if check_mode():
            _check_slots(slot_mapping, nb * bs)
        slots = slot_mapping.data_ptr()
    else:
        _require(block_tables is not None and cache_seqlens is not None,
                 "append needs block_tables and cache_seqlens")
        _table(block_tables, n)
        _require(cache_seqlens.dtype is torch.int32 and cache_seqlens.shape == (n,)
                 and cache_seqlens.is_contiguous(), "cache_seqlens must be contiguous int32 [T]")
        tables, lens, mb = block_tables.data_ptr(), cache_seqlens.data_ptr(), block_tables.shape[1]
    q = torch.empty((n, n_q_heads, HEAD_DIM), dtype=dt, device=qkv.device)
    k = torch.empty((n, hkv, HEAD_DIM), dtype=dt, device=qkv.device) if want_k else None
    _lib.launch("aac_qk_norm_rope_store_kv4", qkv.get_device(), qkv.data_ptr(),
                qkv.stride(0) if n > 1 else qkv.shape[1], n, n_q_heads, hkv, HEAD_DIM,
                q_norm_weight.data_ptr(), k_norm_weight.data_ptr(), float(eps), cos.data_ptr(),
                sin.data_ptr(), cos.shape[0], positions.data_ptr(), q.data_ptr(),
                None if k is None else k.data_ptr(), kv_cache.data_ptr(), nb, bs, slots, tables, mb, lens,
                _code(dt))
    return q, k


def kv4_export(storage: torch.Tensor, block_table, length: int,
               dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The first ``length`` tokens of one sequence in every layer of ``storage`` (``[n_layers,
    num_blocks, Hkv, 2, block_size * 68]``): K and V ``[n_layers, length, Hkv, 128]`` in
    ``dtype`` (bf16 and fp32 hold every value of the cache exactly), zeros where a block is
    outside the pool."""
    k, v = kv4_load(storage.flatten(0, 1), _layer_slots(storage, block_table, length), dtype)
    return k.unflatten(0, (storage.shape[0], length)), v.unflatten(0, (storage.shape[0], length))


def kv4_import(k: torch.Tensor, v: torch.Tensor, storage: torch.Tensor, block_table) -> None:
    """The reverse of ``kv4_export``: quantises ``k`` and ``v`` ``[n_layers, length, Hkv, 128]``
    into the sequence's blocks; those outside the pool are skipped (``IndexError`` for them
    with ``AAC_CHECK=1``).  Rows exported in bf16 or fp32 come back as they were held, byte
    for byte."""
    _require(k.dim() == 4 and k.shape == v.shape and k.shape[0] == storage.shape[0],
             "k and v must be [n_layers, length, Hkv, 128]")
    kv4_store(k.flatten(0, 1), v.flatten(0, 1), storage.flatten(0, 1),
              _layer_slots(storage, block_table, k.shape[1]))


def _layer_slots(storage: torch.Tensor, block_table, length: int) -> torch.Tensor:
    """Rows of the sequence in each layer of the storage taken as one cache; -1 where the
    block is outside the pool."""
    _require(storage.dim() == 5 and storage.is_contiguous(),
             "KV storage must be contiguous [n_layers, num_blocks, Hkv, 2, block_size * 68]")
    nb, bs, _ = _cache(storage[0])
    table = torch.as_tensor(block_table, device=storage.device).reshape(-1).long()
    _require(0 <= length <= table.numel() * bs, "the block table is too short for the length")
    at = torch.arange(length, device=storage.device)
    blk = table[at // bs]
    row = torch.where((blk >= 0) & (blk < nb), blk * bs + at % bs, -1)
    first = torch.arange(storage.shape[0], device=storage.device)[:, None] * (nb * bs)
    return torch.where(row >= 0, first + row, -1).reshape(-1)


@functools.lru_cache(maxsize=4096)
def _ws_bytes(*args: int) -> int:
    """aac_kv4_decode_workspace_bytes: host arithmetic on its integer arguments."""
    return _lib.lib().aac_kv4_decode_workspace_bytes(*args)


def _decode(q, q_stride, n, hq, kv_cache, cache, tables, lens, k, v, ks, vs, scale, mcl, part, out,
            out_stride):
    nb, bs, hkv = cache
    mb = tables.shape[1]
    nbytes = _ws_bytes(n, hq, hkv, HEAD_DIM, bs, mb, mcl, part)
    # From the allocator, in stream order: a captured call's belongs to its graph.  Held until
    # the library has returned, since other threads run while it enqueues its launches.
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _lib.launch("aac_kv4_decode", q.get_device(), q.data_ptr(), q_stride, k, v, ks, vs,
                kv_cache.data_ptr(), nb, bs, tables.data_ptr(), mb, lens.data_ptr(), n, mcl, hq, hkv,
                HEAD_DIM, scale, out.data_ptr(), out_stride, None if ws is None else ws.data_ptr(), nbytes,
                part, _code(q.dtype))


def _heads(hq: int, hkv: int, d: int) -> None:
    if d != HEAD_DIM:
        raise RuntimeError(f"head_dim must be {HEAD_DIM}")
    if hkv == 0 or hq % hkv or hq // hkv > 16:
        raise RuntimeError("query heads must be 1 to 16 times the KV heads")


def _table(block_tables, n: int) -> None:
    if (block_tables.dtype is not torch.int32 or block_tables.dim() != 2
            or block_tables.shape[0] != n or block_tables.shape[1] == 0
            or not block_tables.is_contiguous()):
        raise RuntimeError("block_tables must be contiguous int32 [B, max_blocks]")


def decode_paged_kv4(q: torch.Tensor, kv_cache: torch.Tensor, block_tables: torch.Tensor,
                     context_lens: torch.Tensor, softmax_scale: Optional[float] = None,
                     max_context_len: Optional[int] = None, partition_tokens: int = 0,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``decode_paged`` over the 4-bit cache: ``q [B, Hq, 128]`` (bf16, fp16 or fp32)
    against the first ``context_lens[b]`` tokens of each sequence, in the values that
    the cache stands for; a sequence of none gets zeros.  1 to 16 query heads a KV head."""
    _on_gpu(q, kv_cache, block_tables, context_lens, out)
    cache = _cache(kv_cache)
    if q.dim() != 3:
        raise RuntimeError("q must be [B, Hq, 128]")
    n, hq, d = q.shape
    _heads(hq, cache[2], d)
    qst = q.stride()
    if qst[2] != 1 or qst[1] != d:
        raise RuntimeError("q heads/head_dim must be contiguous")
    _table(block_tables, n)
    if (context_lens.dtype is not torch.int32 or context_lens.shape != (n,)
            or not context_lens.is_contiguous()):
        raise RuntimeError("context_lens must be contiguous int32 [B]")
    row = hq * d
    if out is None:
        out, ost = torch.empty((n, hq, d), dtype=q.dtype, device=q.device), row
    else:
        st = out.stride()
        if out.shape != q.shape or out.dtype is not q.dtype or st[2] != 1 or st[1] != d:
            raise RuntimeError("out must be [B, Hq, 128] like q")
        ost = st[0] if n > 1 else row
    _decode(q, qst[0] if n > 1 else row, n, hq, kv_cache, cache, block_tables, context_lens, None, None, 0,
            0, _scale(softmax_scale, d), min(int(max_context_len or 0), 0x7fffffff), int(partition_tokens), out, ost)
    return out


def flash_attn_with_kv4cache(q: torch.Tensor, kv_cache: torch.Tensor,
                             k: Optional[torch.Tensor] = None, v: Optional[torch.Tensor] = None, *,
                             cache_seqlens: torch.Tensor | int, block_table: torch.Tensor,
                             softmax_scale: Optional[float] = None, causal: bool = False,
                             num_splits: int = 0,
                             max_context_len: Optional[int] = None) -> torch.Tensor:
    """``flash_attn_with_kvcache`` over the 4-bit cache: ``q [B, 1, Hq, 128]``; ``k``/``v``
    (``[B, 1, Hkv, 128]``), where given, are quantised into the cache at position
    ``cache_seqlens[b]`` and the call attends over ``cache_seqlens[b] + 1`` tokens,
    otherwise over ``cache_seqlens[b]`` (int32 ``[B]``, or an int for all).  The new token
    is attended to as the cache holds it.  All rows are written before any is read;
    ``cache_seqlens`` is not modified.  ``causal`` changes nothing for one query token;
    ``num_splits``, where positive, is how many partitions the longest context is split into
    at most (of a multiple of 256 tokens)."""
    if q.dim() != 4:
        raise RuntimeError("q must be [B, S, Hq, 128]")
    n, s, hq, d = q.shape
    if s != 1:
        raise NotImplementedError("only one query token per sequence (decode) is supported")
    if (k is None) != (v is None):
        raise RuntimeError("k and v must be given together")
    if isinstance(cache_seqlens, int):
        _on_gpu(q, kv_cache, k, v, block_table)
        cache_seqlens = torch.full((n,), cache_seqlens, dtype=torch.int32, device=q.device)
    else:
        _on_gpu(q, kv_cache, k, v, cache_seqlens, block_table)
        cache_seqlens = cache_seqlens.contiguous()
    cache = _cache(kv_cache)
    hkv = cache[2]
    _heads(hq, hkv, d)
    block_table = block_table.contiguous()
    _table(block_table, n)
    if cache_seqlens.dtype is not torch.int32 or cache_seqlens.shape != (n,):
        raise RuntimeError("cache_seqlens must be int32 [B]")
    qst = q.stride()
    if qst[3] != 1 or qst[2] != d:
        q = q.contiguous()
        qst = q.stride()
    out = torch.empty((n, 1, hq, d), dtype=q.dtype, device=q.device)
    kp = vp = None
    ks = vs = 0
    if k is not None:
        if k.shape != v.shape or k.shape != (n, 1, hkv, d):
            raise RuntimeError("k/v must be [B, 1, Hkv, 128]")
        if k.dtype is not q.dtype or v.dtype is not q.dtype:
            raise RuntimeError("k/v dtype mismatch")
        kst, vst = k.stride(), v.stride()
        if kst[3] != 1 or kst[2] != d:
            k = k.contiguous()
            kst = k.stride()
        if vst[3] != 1 or vst[2] != d:
            v = v.contiguous()
            vst = v.stride()
        row = hkv * d
        kp, vp = k.data_ptr(), v.data_ptr()
        ks, vs = (kst[0], vst[0]) if n > 1 else (row, row)
    row = hq * d
    most = min(int(max_context_len or 0), 0x7fffffff)
    part = 0
    if num_splits and num_splits > 0:
        cap = min(block_table.shape[1] * cache[1], 0x7fffffff)
        part = -(-(min(most, cap) if most > 0 else cap) // int(num_splits))
    _decode(q, qst[0] if n > 1 else row, n, hq, kv_cache, cache, block_table, cache_seqlens, kp, vp, ks, vs,
            _scale(softmax_scale, d), most, part, out, row)
    return out
