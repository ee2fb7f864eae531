"""Rotary positions: the rotation of query and key heads by their tokens' angles, alone
(``apply_rotary_emb``) or on the way into the paged KV cache (``rotary_append_paged``,
``flash_attn_with_kvcache(rotary_cos=...)``), and the tables of cos and sin, scaled for
long contexts where a model's configuration says so (``RotaryEmbedding``).

The first ``R`` dims of a head are ``R / 2`` pairs, ``(d, d + R / 2)`` or, interleaved,
``(2 d, 2 d + 1)``; ``cos`` and ``sin`` are ``[positions, R / 2]``, in the heads' type or
float32.  The rotation is computed in float32 and rounded once; dims from ``R`` on pass
unchanged.  A position outside the tables takes their first or last row.  As everywhere
here: ``RuntimeError`` for a rejected argument, the current stream, no synchronisation, no
gradients."""
from __future__ import annotations

import math
from typing import Optional, Union

import torch

from . import _lib
from .flash_attn_interface import _on_gpu, _require

__all__ = ["apply_rotary_emb", "rotary_append_paged", "RotaryEmbedding", "scaled_frequencies"]


_CODES = _lib.AAC_DTYPE
_DENSE = torch.contiguous_format


def _bad_dtype(dtype):
    raise RuntimeError(f"unsupported dtype {dtype}")


# (A call's host time is its latency for a single token: one condition a line, messages
# built where they are raised.)
def _tables(cos: torch.Tensor, sin: torch.Tensor, dtype: torch.dtype, head_dim: int):
    """(cos, sin addresses, rows, rotary dims, type code) of the tables, checked."""
    shape = cos.shape
    if len(shape) != 2 or sin.shape != shape or not cos.is_contiguous() or not sin.is_contiguous():
        raise RuntimeError("cos and sin must be contiguous [positions, rotary_dim / 2]")
    td = cos.dtype
    if sin.dtype is not td or (td is not dtype and td is not torch.float32):
        raise RuntimeError("cos and sin must be float32 or of the heads' dtype")
    rows, half = shape
    if rows == 0 or half == 0:
        raise RuntimeError("empty tables")
    if 2 * half > head_dim:
        raise RuntimeError("rotary_dim is larger than head_dim")
    return cos.data_ptr(), sin.data_ptr(), min(rows, (1 << 31) - 1), 2 * half, _CODES.get(td)


def _ints(t: torch.Tensor, n: int, name: str) -> int:
    """The address of an int32 vector, checked."""
    if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous int32 [{n}]")
    return t.data_ptr()


def _strides(t: torch.Tensor):
    """(sequence, token, head) strides of [B, S, H, D] or, with 0 first, [N, H, D]."""
    st = t.stride()
    if st[-1] != 1 and t.shape[-1] != 1:
        raise RuntimeError("head_dim must be contiguous")
    return st[:3] if len(st) == 4 else (0, st[0], st[1])


def apply_rotary_emb(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool = False,
                     inplace: bool = False, seqlen_offsets: Union[int, torch.Tensor] = 0,
                     cu_seqlens: Optional[torch.Tensor] = None, max_seqlen: Optional[int] = None, *,
                     conjugate: bool = False) -> torch.Tensor:
    """The heads of ``x`` turned by their tokens' angles.

    x ``[B, S, H, D]``: token ``i`` of sequence ``b`` stands at ``seqlen_offsets + i`` (an
    int, or int32 ``[B]``).  With ``cu_seqlens`` (int32 ``[B + 1]``) x is packed
    ``[N, H, D]``, sequence ``b`` rows ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]``; rows of no
    sequence are left as they are in place, and undefined in a new output; ``max_seqlen``
    is not needed.  Any strides whose last is 1.  ``conjugate`` turns back (the inverse).
    Returns a new contiguous tensor, or ``x`` itself with ``inplace``.  bf16, fp16 and
    float32, any even head_dim."""
    dev = x.get_device()
    if dev < 0 or cos.get_device() != dev or sin.get_device() != dev:
        _on_gpu(x, cos, sin)
    shape = x.shape
    if len(shape) != (4 if cu_seqlens is None else 3):
        raise RuntimeError("x must be [tokens, heads, head_dim] with cu_seqlens, [B, S, heads, head_dim] without")
    D = shape[-1]
    if D % 2:
        raise RuntimeError("head_dim must be even")
    if cu_seqlens is not None:
        _on_gpu(x, cu_seqlens)
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
            raise RuntimeError("cu_seqlens must be [B + 1]")
        B, S, N = cu_seqlens.shape[0] - 1, 0, shape[0]
        cu = _ints(cu_seqlens, B + 1, "cu_seqlens")
    else:
        B, S = shape[0], shape[1]
        N, cu = 0, None
    if isinstance(seqlen_offsets, torch.Tensor):
        if seqlen_offsets.get_device() != dev:
            _on_gpu(x, seqlen_offsets)
        offset, offsets = 0, _ints(seqlen_offsets, B, "seqlen_offsets")
    else:
        offset, offsets = int(seqlen_offsets), None
        if not -(1 << 31) <= offset < 1 << 31:
            raise RuntimeError("seqlen_offsets does not fit in 32 bits")
    dt = x.dtype
    cp, sp, rows, rot, tcode = _tables(cos, sin, dt, D)
    code = _CODES.get(dt)
    if code is None:
        _bad_dtype(dt)
    s0, s1, s2 = _strides(x)
    if inplace:
        out, (o0, o1, o2) = x, (s0, s1, s2)
        for n, s in zip(shape, x.stride()):
            if s == 0 and n > 1:
                raise RuntimeError("x is broadcast: it cannot be turned in place")
    else:
        out = torch.empty_like(x, memory_format=_DENSE)
        o2 = D
        o1 = shape[-2] * D
        o0 = S * o1
    if x.numel() and B:
        _lib.launch("aac_rotary", dev, x.data_ptr(), s0, s1, s2, out.data_ptr(), o0, o1, o2, B, S, N, cu,
                    offsets, offset, shape[-2], D, cp, sp, rows, rot, 1 if interleaved else 0,
                    1 if conjugate else 0, tcode, code)
    return out


def _append(q, k, v, k_cache, v_cache, tables, seqlens, cos, sin, interleaved, cu, q_at_first, ctx=None):
    """The launch of ``rotary_append_paged``; shapes of q, k, v and tables checked there."""
    nblk, bs, hkv, D = k_cache.shape
    dt = k.dtype
    cp, sp, rows, rot, tcode = (None, None, 0, 0, 0) if cos is None else _tables(cos, sin, dt, D)
    code = _CODES.get(dt)
    if code is None:
        _bad_dtype(dt)
    B = seqlens.shape[0]
    if cu is None:
        sk, n = k.shape[1], 0
    else:
        sk, n, cu = 0, k.shape[0], cu.data_ptr()
    k0, k1, k2 = _strides(k)
    v0, v1, v2 = _strides(v)
    out = qp = qo = None
    q0 = q1 = q2 = sq = hq = 0
    if q is not None:
        out = torch.empty_like(q, memory_format=_DENSE)
        q0, q1, q2 = _strides(q)
        qp, qo, hq = q.data_ptr(), out.data_ptr(), q.shape[-2]
        if cu is None:
            sq = q.shape[1]
    if B and (k.numel() or (q is not None and q.numel())):
        kc = k_cache.data_ptr()
        _lib.launch("aac_rotary_append_paged", k.get_device(), qp, q0, q1, q2, k.data_ptr() or kc, k0, k1, k2,
                    v.data_ptr() or kc, v0, v1, v2, qo, B, sq, sk, n, cu, seqlens.data_ptr(),
                    None if ctx is None else ctx.data_ptr(), hq, hkv, D, cp, sp, rows, rot,
                    1 if interleaved else 0, 1 if q_at_first else 0, kc, v_cache.data_ptr(), nblk, bs,
                    tables.data_ptr(), tables.shape[1], tcode, code)
    return out


def rotary_append_paged(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor,
                        k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                        cache_seqlens: torch.Tensor, rotary_cos: Optional[torch.Tensor] = None,
                        rotary_sin: Optional[torch.Tensor] = None, *, interleaved: bool = False,
                        cu_seqlens: Optional[torch.Tensor] = None,
                        max_seqlen: Optional[int] = None) -> Optional[torch.Tensor]:
    """Append new tokens to a paged cache, their keys turned by their positions on the way,
    and return their queries turned alike (None for ``q`` None).

    New token ``i`` of sequence ``b`` stands at ``cache_seqlens[b] + i`` (int32 ``[B]``, not
    modified) and goes to the row ``block_tables`` (int32 ``[B, max_blocks]``) names for
    that position in the caches ``[num_blocks, block_size, Hkv, D]``; one without a block
    is skipped, as ``flash_attn_with_kvcache`` skips it.  q ``[B, S, Hq, D]``, k and v
    ``[B, S, Hkv, D]``, or, with ``cu_seqlens`` (int32 ``[B + 1]``), packed ``[N, ..., D]``
    (rows of no sequence: not stored, their queries undefined; ``max_seqlen`` is not
    needed).  Any strides whose last is 1: they may be views of the fused projection.
    Without ``rotary_cos`` / ``rotary_sin`` nothing is turned (q is copied).  Rows are
    distinct: of two tokens for one row an unspecified one stays.  bf16, fp16, float32, any
    even head_dim."""
    _on_gpu(q, k, v, k_cache, v_cache, block_tables, cache_seqlens, rotary_cos, rotary_sin, cu_seqlens)
    if (rotary_cos is None) != (rotary_sin is None):
        raise RuntimeError("rotary_cos and rotary_sin go together")
    cshape, kshape = k_cache.shape, k.shape
    if (len(cshape) != 4 or cshape != v_cache.shape or not k_cache.is_contiguous()
            or not v_cache.is_contiguous()):
        raise RuntimeError("caches must be contiguous [num_blocks, block_size, Hkv, D], alike")
    nd = 4 if cu_seqlens is None else 3
    if len(kshape) != nd or kshape != v.shape or kshape[-2:] != cshape[2:]:
        raise RuntimeError("k and v must be [B, S, Hkv, D], or [N, Hkv, D] with cu_seqlens, as the caches' rows")
    dt = k.dtype
    if v.dtype is not dt or k_cache.dtype is not dt or v_cache.dtype is not dt:
        raise RuntimeError("dtype mismatch")
    D = cshape[3]
    if D % 2 or 0 in cshape:
        raise RuntimeError("head_dim must be even, the caches not empty")
    if q is not None and (q.dim() != nd or q.dtype is not dt or q.shape[-1] != D
                          or q.shape[:nd - 2] != kshape[:nd - 2]):
        raise RuntimeError("q must be [B, S, Hq, D], or [N, Hq, D], of k's tokens and dtype")
    B = cache_seqlens.shape[0] if cache_seqlens.dim() == 1 else -1
    _ints(cache_seqlens, B, "cache_seqlens")
    if cu_seqlens is not None:
        _ints(cu_seqlens, B + 1, "cu_seqlens")
    elif kshape[0] != B:
        raise RuntimeError("cache_seqlens must be [B]")
    tshape = block_tables.shape
    if (block_tables.dtype is not torch.int32 or len(tshape) != 2 or tshape[0] != B or tshape[1] == 0
            or not block_tables.is_contiguous()):
        raise RuntimeError("block_tables must be contiguous int32 [B, max_blocks]")
    return _append(q, k, v, k_cache, v_cache, block_tables, cache_seqlens, rotary_cos, rotary_sin,
                   interleaved, cu_seqlens, False)


# ------------------------------------------------------------------ frequencies and tables
def scaled_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: Optional[dict] = None,
                       seq_len: Optional[int] = None) -> tuple[torch.Tensor, float]:
    """(float64 ``[rotary_dim / 2]`` radians a position, the factor of cos and sin).

    Unscaled: ``theta ** (-2 i / rotary_dim)``.  ``scaling`` is the rule a model's
    configuration holds (``rope_scaling``), by its ``rope_type`` (or ``type``):

    * ``linear``: positions divided by ``factor``;
    * ``dynamic``: theta grown for a context of ``seq_len`` tokens past
      ``original_max_position_embeddings``, with ``factor``;
    * ``yarn``: frequencies of more than ``beta_fast`` (32) turns in the original context
      kept, of fewer than ``beta_slow`` (1) divided by ``factor``, a ramp between (its ends
      whole dims unless ``truncate`` is false), and cos and sin times ``attention_factor``
      (``0.1 ln(factor) + 1``, or from ``mscale`` and ``mscale_all_dim``);
    * ``llama3``: frequencies of more than ``high_freq_factor`` turns kept, of fewer than
      ``low_freq_factor`` divided by ``factor``, between them in proportion."""
    _require(rotary_dim > 0 and rotary_dim % 2 == 0, "rotary_dim must be positive and even")
    _require(theta > 1, "theta must be above 1")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    inv = float(theta) ** (-i / rotary_dim)
    if not scaling:
        return inv, 1.0
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "default":
        return inv, 1.0

    def need(*names):
        for n in names:
            _require(scaling.get(n) is not None, f"rope scaling {kind!r} needs {n!r}")
        return [float(scaling[n]) for n in names]

    factor, = need("factor")
    _require(factor >= 1, "the scaling's factor must be 1 or more")
    if kind == "linear":
        return inv / factor, 1.0
    old, = need("original_max_position_embeddings")
    _require(old > 0, "original_max_position_embeddings must be positive")
    if kind == "dynamic":
        _require(rotary_dim > 2, "dynamic scaling needs more than one frequency")
        n = float(seq_len or 0)
        if n > old:
            grown = float(theta) * (factor * n / old - (factor - 1)) ** (rotary_dim / (rotary_dim - 2))
            inv = grown ** (-i / rotary_dim)
        return inv, 1.0
    if kind == "yarn":
        fast, slow = float(scaling.get("beta_fast") or 32), float(scaling.get("beta_slow") or 1)

        def dim_of(turns):  # the dim that makes so many turns in the original context
            return rotary_dim * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo, hi = dim_of(fast), dim_of(slow)
        if scaling.get("truncate", True):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, rotary_dim - 1)
        ramp = ((i / 2 - lo) / (hi - lo if hi != lo else 0.001)).clamp(0, 1)
        att = scaling.get("attention_factor")
        if att is None:
            def size(m):
                return 0.1 * m * math.log(factor) + 1

            a, b = scaling.get("mscale"), scaling.get("mscale_all_dim")
            att = size(float(a)) / size(float(b)) if a and b else size(1.0)
        return inv / factor * ramp + inv * (1 - ramp), float(att)
    if kind == "llama3":
        lo, hi = need("low_freq_factor", "high_freq_factor")
        _require(hi > lo, "high_freq_factor must be above low_freq_factor")
        keep = ((old * inv / (2 * math.pi) - lo) / (hi - lo)).clamp(0, 1)
        return inv / factor * (1 - keep) + inv * keep, 1.0
    raise RuntimeError(f"unknown rope scaling {kind!r}: linear, dynamic, yarn or llama3")


class RotaryEmbedding:
    """The frequencies of a model's rotary positions (``scaled_frequencies``), held on a
    GPU, and the tables built from them."""

    def __init__(self, rotary_dim: int, theta: float = 10000.0, scaling: Optional[dict] = None, *,
                 seq_len: Optional[int] = None, device="cuda"):
        self.rotary_dim = rotary_dim
        self.frequencies, self.factor = scaled_frequencies(rotary_dim, theta, scaling, seq_len)
        self.device = torch.device(device)
        _require(self.device.type == "cuda", "the tables are built on a GPU (no CPU path exists)")
        self._turns = (self.frequencies / (2 * math.pi)).to(self.device)
        self.device = self._turns.device

    def cos_sin(self, n: Optional[int] = None, *, start: int = 0,
                positions: Optional[torch.Tensor] = None,
                dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
        """cos and sin, times the scaling's factor, ``[n, rotary_dim / 2]`` of positions
        ``start`` to ``start + n - 1``, or of ``positions`` (int32 ``[n]`` on the GPU).
        Angles are reduced in 64 bits: far positions lose nothing."""
        code = _CODES.get(dtype)
        if code is None:
            _bad_dtype(dtype)
        dev, at = self._turns.get_device(), None
        if positions is not None:
            if n is not None or start:
                raise RuntimeError("positions, or n and start")
            if positions.dim() != 1 or positions.get_device() != dev:
                raise RuntimeError("positions must be one-dimensional, on the tables' GPU")
            n = positions.shape[0]
            at = _ints(positions, n, "positions")
        if n is None or n < 0:
            raise RuntimeError("n must be given, 0 or more")
        if abs(start) > 1 << 40:  # (here, before it is cut to 64 bits)
            raise RuntimeError("inconsistent arguments: start is past 2^40")
        half = self.rotary_dim // 2
        cos = torch.empty((n, half), dtype=dtype, device=self.device)
        sin = torch.empty_like(cos)
        if n:
            _lib.launch("aac_rotary_tables", dev, self._turns.data_ptr(), half, at, int(start), n, self.factor,
                        cos.data_ptr(), sin.data_ptr(), code)
        return cos, sin
