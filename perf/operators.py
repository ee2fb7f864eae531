"""The measured operators: serving with a KV cache held in four bits.

Each case is one pass through one operator (or the pair a user calls together),
over the range of sizes the serving engine is used at:

* ``store``    -- ``kv4.kv4_store`` quantises packed K/V rows into the paged 4-bit
  cache and ``kv4.kv4_load`` reads them back, as a migration of the request does;
* ``attend``   -- ``kv4.decode_paged_kv4``: one query token a sequence over the cache;
* ``append``   -- ``kv4.flash_attn_with_kv4cache``: append the new token, attend, and
  ``kv4_load`` of the appended rows;
* ``maps``     -- ``paged.build_step_maps``: block tables, slot mapping, positions and
  cu_seqlens of a step from its request lengths, on the GPU;
* ``logprobs`` -- ``fused.token_logprobs``: log probability of given tokens, entropy and
  the top alternatives of each row of logits.

The 4-bit cache is uint8 ``[num_blocks, Hkv, 2, block_size * 68]``: for each block and
KV head the K page, then the V page; a page is ``block_size`` rows of 64 bytes (dim
``2 i`` in the low nibble of byte ``i``, E2M1) and then ``block_size`` rows of 4 scale
bytes (E8M0, one for 32 dims).

``run`` makes the framework's calls where ``own`` is true and computes the same with
elementary torch operations where it is not.  Lengths come from the case itself
(``lens_seed``), values from ``prepare``'s seed.  ``exact`` recomputes a case in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

D = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MAX_STORE_TOKENS = 262144      # of the largest listed store, at 8 KV heads in 16 bits
MAX_KV_TOKENS = 1600000        # cached tokens of the largest listed attention, at 8 KV heads
MAX_LOGIT_BYTES = 1200000000   # of the largest listed call


def listed():
    return [
        # one newly admitted request of odd length, some of its rows padding
        dict(name="store_fp16_777", kind="store", dtype="fp16", tokens=777, hkv=8, block=16,
             pad=0.1),
        # the engine's largest prefill: 256 prompts of 1024 tokens, one layer
        dict(name="store_262144", kind="store", dtype="bf16", tokens=262144, hkv=8, block=256,
             pad=0.0),
        # the smallest attention: a handful of sequences in fp32; latency is what counts
        dict(name="attend_fp32_4", kind="attend", dtype="fp32", seqs=4, lo=17, hi=511, hq=16,
             hkv=8, block=256, lens_seed=1),
        # a lightly loaded server's decode step: append and attend, small blocks
        dict(name="append_24", kind="append", dtype="bf16", seqs=24, lo=100, hi=2063, hq=16,
             hkv=8, block=16, lens_seed=2),
        # the headline decode step: 256 sequences of 1-2k tokens
        dict(name="attend_256", kind="attend", dtype="bf16", seqs=256, lo=1024, hi=2047, hq=16,
             hkv=8, block=256, lens_seed=3),
        # long contexts with four query heads per KV head: the keys are split
        dict(name="attend_long_64", kind="attend", dtype="bf16", seqs=64, lo=16384, hi=32768,
             hq=32, hkv=8, block=256, lens_seed=4),
        # one very long request in fp16, eight query heads per KV head
        dict(name="attend_one_fp16", kind="attend", dtype="fp16", seqs=1, lo=100001, hi=131071,
             hq=64, hkv=8, block=64, lens_seed=5),
        # a decode step's maps: one token a sequence, some of them need a new block
        dict(name="maps_decode_24", kind="maps", seqs=24, lo=1, hi=1, cached=2063, block=16,
             width=144, slack=0, lens_seed=6),
        # the largest prefill's maps: every block is new
        dict(name="maps_prefill_256", kind="maps", seqs=256, lo=1024, hi=1024, cached=0,
             block=256, width=9, slack=0, lens_seed=7),
        # one interactive user who asks for five alternatives
        dict(name="logprobs_1", kind="logprobs", dtype="bf16", rows=1, cols=151936, top=5,
             allowed=0),
        # the 256-sequence step with the most alternatives an API offers
        dict(name="logprobs_256", kind="logprobs", dtype="bf16", rows=256, cols=151936, top=20,
             allowed=0),
        # scoring prompts: thousands of rows whose length breaks their alignment
        dict(name="logprobs_3900", kind="logprobs", dtype="fp16", rows=3900, cols=151937, top=1,
             allowed=0),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random) -> dict:
    """One more case of the ranges above."""
    kind = rng.choice(["store", "attend", "attend", "append", "maps", "logprobs", "logprobs"])
    seed = rng.randrange(1 << 30)
    if kind == "store":
        dtype, hkv = rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice([1, 4, 8, 8])
        return dict(kind=kind, dtype=dtype, hkv=hkv, block=rng.choice([16, 48, 64, 256]),
                    tokens=_log_int(rng, 1, MAX_STORE_TOKENS // (2 if dtype == "fp32" else 1)),
                    pad=rng.choice([0.0, 0.0, 0.3]))
    if kind in ("attend", "append"):
        hq, hkv = rng.choice([(16, 8), (16, 8), (32, 8), (8, 4), (8, 8), (48, 4), (7, 1), (64, 8)])
        seqs = _log_int(rng, 1, 256)
        most = min(131071, MAX_KV_TOKENS * 3 // 4 // seqs)
        hi = _log_int(rng, 16, max(17, most))
        return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), seqs=seqs,
                    lo=rng.choice([0, rng.randint(1, hi), rng.randint(1, hi)]), hi=hi, hq=hq,
                    hkv=hkv, block=rng.choice([16, 48, 64, 256]), lens_seed=seed)
    if kind == "maps":
        seqs = _log_int(rng, 1, 1000)
        hi = rng.choice([1, _log_int(rng, 1, MAX_STORE_TOKENS // seqs)])
        cached = rng.choice([0, rng.randint(1, 3000)])
        block = rng.choice([16, 48, 64, 256])
        return dict(kind=kind, seqs=seqs, lo=rng.randint(0, hi), hi=hi, cached=cached, block=block,
                    width=-(-(hi + cached) // block) + rng.randint(0, 3),
                    slack=rng.choice([0, 0, 37]), lens_seed=seed)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    cols = rng.choice([2048, 32000, 50257, 151936, 151937])
    most = MAX_LOGIT_BYTES // (cols * (4 if dtype == "fp32" else 2))
    return dict(kind=kind, dtype=dtype, rows=_log_int(rng, 1, min(4096, most)), cols=cols,
                top=rng.choice([0, 1, 5, 20, rng.randint(0, 32)]), allowed=rng.choice([0, 0, 3, 400]))


# ------------------------------------------------------------------ helpers
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _lens(case) -> list[int]:
    r = random.Random(case["lens_seed"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]


def _channels(g, hkv):
    """A key's channels differ in size, a few of them by much, in a trained model."""
    c = torch.exp(0.4 * _randn(g, hkv, D))
    c[:, torch.randint(0, D, (4,), generator=g, device="cuda")] *= 6.0
    return c


# ------------------------------------------------------------------ the 4-bit format
def _quantise(x):
    """float32 ``[..., D]`` -> (codes uint8 ``[..., D / 2]``, scales uint8 ``[..., D / 32]``)."""
    x = x.reshape(*x.shape[:-1], -1, 32)
    a = x.abs().amax(-1)
    # the exponent of a rounded to two significant bits, less that of the largest code
    e = ((a.view(torch.int32) + 0x200000) >> 23) - 127 - 2
    e = e.clamp(-125, 125)
    y = torch.ldexp(x.abs(), -e.unsqueeze(-1))
    y = torch.where(y < 2, torch.round(y * 2) / 2, torch.where(y < 4, torch.round(y),
                                                             torch.round(y / 2) * 2)).clamp_(max=6.0)
    code = torch.where(y < 2, y * 2, torch.where(y < 4, y + 2, y / 2 + 4)).to(torch.uint8)
    code += (x < 0).to(torch.uint8) * 8
    bad = ~torch.isfinite(a)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code).flatten(-2)
    scale = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return code[..., ::2] | (code[..., 1::2] << 4), scale


def _values(codes, scales):
    """The float32 values that codes and scales stand for."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0,
                          -3.0, -4.0, -6.0], device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    x = table[both.int()].unflatten(-1, (-1, 32))
    size = torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127)
    size = torch.where(scales == 255, torch.full_like(size, math.nan), size)
    return (x * size.unsqueeze(-1)).flatten(-2)


def _pages(cache, block):
    """(K codes, K scales, V codes, V scales) of a cache: views ``[blocks, Hkv, block, 64 | 4]``."""
    out = []
    for i in range(2):
        page = cache[:, :, i]
        out.append(page[..., :block * 64].unflatten(-1, (block, 64)))
        out.append(page[..., block * 64:].unflatten(-1, (block, 4)))
    return out


def _put(cache, block, slots, k, v):
    keep = slots >= 0
    blk, row = slots[keep] // block, slots[keep] % block
    for i, x in enumerate((k, v)):
        codes, scales = _quantise(x[keep].float())
        pages = _pages(cache, block)
        pages[2 * i][blk, :, row] = codes
        pages[2 * i + 1][blk, :, row] = scales


def _get(cache, block, slots, dtype):
    blk, row = slots.clamp(min=0) // block, slots.clamp(min=0) % block
    kc, ks, vc, vs = _pages(cache, block)
    none = (slots < 0)[:, None, None]
    return tuple(_values(c[blk, :, row], s[blk, :, row]).masked_fill(none, 0.0).to(dtype)
                 for c, s in ((kc, ks), (vc, vs)))


# ------------------------------------------------------------------ store
def _prepare_store(case, seed):
    g, n, hkv, bs = _gen(seed), case["tokens"], case["hkv"], case["block"]
    dt = DTYPES[case["dtype"]]
    # k is the normalised and rotated copy, v a view of the QKV projection's output
    # (as wide as two query heads a KV head make it, where that is not too large)
    k = (_randn(g, n, hkv, D) * _channels(g, hkv)).to(dt)
    wide = 4 if n <= 65536 else 2
    v = _randn(g, n, wide * hkv * D, dtype=dt)[:, (wide - 1) * hkv * D:].view(n, hkv, D)
    blocks = -(-n // bs) + 1
    order = torch.randperm(blocks, generator=g, device="cuda")
    i = torch.arange(n, device="cuda")
    slots = order[i // bs] * bs + i % bs
    if case["pad"]:
        slots[torch.rand(n, generator=g, device="cuda") < case["pad"]] = -1
    cache = torch.zeros((blocks, hkv, 2, bs * 68), dtype=torch.uint8, device="cuda")
    return dict(k=k, v=v, slots=slots, cache=cache, block=bs, dtype=dt)


def _run_store(s):
    if own:
        from awesome_acceleration_amd import kv4
        kv4.kv4_store(s["k"], s["v"], s["cache"], s["slots"])
        k, v = kv4.kv4_load(s["cache"], s["slots"], dtype=s["dtype"])
    else:
        _put(s["cache"], s["block"], s["slots"], s["k"], s["v"])
        k, v = _get(s["cache"], s["block"], s["slots"], s["dtype"])
    return {"k": k, "v": v}


def _held(x):
    """What the cache stands for after a store of ``x``, from the format's definition in 64 bits."""
    x = x.double().reshape(*x.shape[:-1], D // 32, 32)
    a = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(a)                               # a = m 2^e, 0.5 <= m < 1
    e = (e - 3 + (m >= 0.875).to(e.dtype)).clamp(-125, 125)
    unit = torch.ldexp(torch.ones_like(a), e)
    y = (x / unit).abs()
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    q = torch.zeros_like(y)
    for i in range(1, 8):  # past the midpoint, or on it where the upper code is the even one
        mid = (grid[i - 1] + grid[i]) / 2
        q = torch.where((y >= mid) if i % 2 == 0 else (y > mid), grid[i], q)
    q = torch.where(torch.isfinite(a), torch.copysign(q, x) * unit, torch.full_like(q, math.nan))
    return q.flatten(-2)


def _exact_store(case, seed):
    s = _prepare_store(case, seed)
    none = (s["slots"] < 0)[:, None, None]
    return {x: torch.cat([_held(p).masked_fill_(n, 0.0).to(torch.float32 if case["dtype"] != "fp32"
                                                          else torch.float64)
                          for p, n in zip(s[x].split(32768), none.split(32768))]) for x in "kv"}


# ------------------------------------------------------------------ attention
def _prepare_attend(case, seed):
    lens, dt, bs = _lens(case), DTYPES[case["dtype"]], case["block"]
    g, n, hq, hkv = _gen(seed), case["seqs"], case["hq"], case["hkv"]
    need = [max(1, -(-x // bs)) for x in lens]
    ids = list(range(sum(need)))
    random.Random(seed).shuffle(ids)
    tables = torch.zeros((n, max(need)), dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        tables[b, :m] = torch.tensor(ids[at:at + m], dtype=torch.int32)
        at += m
    cache = torch.empty((len(ids), hkv, 2, bs * 68), dtype=torch.uint8, device="cuda")
    size = _channels(g, hkv)[:, None]
    step = max(1, 65536 // bs)
    for a in range(0, len(ids), step):
        kc, ks, vc, vs = _pages(cache[a:a + step], bs)
        shape = kc.shape[:3]
        kc[:], ks[:] = _quantise(_randn(g, *shape, D) * size)
        vc[:], vs[:] = _quantise(_randn(g, *shape, D))
    s = dict(q=_randn(g, n, hq, D, dtype=dt), cache=cache, tables=tables.cuda(), lens=lens,
             ctx=torch.tensor(lens, dtype=torch.int32, device="cuda"), block=bs, most=max(lens),
             scale=D ** -0.5)
    if case["kind"] == "append":
        # a sequence's new token is the last of its context; one of length zero gets its first
        s["k"] = (_randn(g, n, 1, hkv, D) * size.view(1, 1, hkv, D)).to(dt)
        s["v"] = _randn(g, n, 1, hkv, D, dtype=dt)
        s["lens"] = [max(1, x) for x in lens]
        s["cached"] = (s["ctx"] - 1).clamp_(min=0)
        t = s["cached"].long()
        s["slots"] = s["tables"].gather(1, (t // bs)[:, None])[:, 0].long() * bs + t % bs
        s["most"] = max(s["lens"])
    return s


def _attend(q, cache, tables, lens, block, scale):
    out = torch.zeros(q.shape, dtype=torch.float32, device=q.device)
    kc, ks, vc, vs = _pages(cache, block)
    hkv = kc.shape[1]
    for b, n in enumerate(lens):
        if n == 0:
            continue  # a row without a key is zero
        t = tables[b, :-(-n // block)].long()
        k = _values(kc[t], ks[t]).transpose(0, 1).flatten(1, 2)[:, :n]   # [Hkv, n, D]
        p = torch.matmul(q[b].float().view(hkv, -1, D), k.transpose(1, 2).contiguous()) * scale
        p = torch.exp(p - p.amax(-1, keepdim=True))
        v = _values(vc[t], vs[t]).transpose(0, 1).flatten(1, 2)[:, :n]
        out[b] = (torch.matmul(p, v.contiguous()) / p.sum(-1, keepdim=True)).view(-1, D)
    return out.to(q.dtype)


def _run_attend(s):
    if own:
        from awesome_acceleration_amd import kv4
        return {"out": kv4.decode_paged_kv4(s["q"], s["cache"], s["tables"], s["ctx"],
                                            softmax_scale=s["scale"], max_context_len=s["most"])}
    return {"out": _attend(s["q"], s["cache"], s["tables"], s["lens"], s["block"], s["scale"])}


def _run_append(s):
    n, hq, _ = s["q"].shape
    if own:
        from awesome_acceleration_amd import kv4
        out = kv4.flash_attn_with_kv4cache(s["q"].view(n, 1, hq, D), s["cache"], k=s["k"], v=s["v"],
                                           cache_seqlens=s["cached"], block_table=s["tables"],
                                           softmax_scale=s["scale"], max_context_len=s["most"])
        k, v = kv4.kv4_load(s["cache"], s["slots"], dtype=s["q"].dtype)
    else:
        _put(s["cache"], s["block"], s["slots"], s["k"][:, 0], s["v"][:, 0])
        out = _attend(s["q"], s["cache"], s["tables"], s["lens"], s["block"], s["scale"])
        out = out.view(n, 1, hq, D)
        k, v = _get(s["cache"], s["block"], s["slots"], s["q"].dtype)
    return {"out": out, "k": k, "v": v}


def _exact_attend(case, seed):
    s = _prepare_attend(case, seed)
    bs, hkv = case["block"], case["hkv"]
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")
    grid = torch.cat((grid, -grid))
    pairs = torch.stack((grid.repeat(16), grid.repeat_interleave(16)), -1)   # of each byte

    def rows(pages, i, n):
        part = pages[:, :, i]
        codes = part[:, :, :bs * 64].reshape(-1, hkv, bs, 64)
        scales = part[:, :, bs * 64:].reshape(-1, hkv, bs, 4)
        x = pairs[codes.int()].reshape(-1, hkv, bs, 4, 32)
        x = x * torch.exp2(scales.double() - 127.0)[..., None]
        return x.reshape(-1, hkv, bs, D).transpose(0, 1).reshape(hkv, -1, D)[:, :n]

    new = None
    if case["kind"] == "append":
        new = _held(s["k"][:, 0]), _held(s["v"][:, 0])
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"]):
        if not n:
            continue
        pages = s["cache"][s["tables"][b, :-(-n // bs)].long()]
        k = rows(pages, 0, n)
        if new is not None:
            k[:, n - 1] = new[0][b]
        x = torch.matmul(k, s["q"][b].double().view(hkv, -1, D).transpose(1, 2).contiguous())
        del k
        p = torch.softmax(x * s["scale"], 1).transpose(1, 2).contiguous()
        v = rows(pages, 1, n)
        if new is not None:
            v[:, n - 1] = new[1][b]
        out[b] = torch.matmul(p, v).reshape(-1, D)
    if new is None:
        return {"out": out}
    return {"out": out[:, None], "k": new[0], "v": new[1]}


# ------------------------------------------------------------------ maps
def _prepare_maps(case, seed):
    r = random.Random(case["lens_seed"])
    n, bs, w = case["seqs"], case["block"], case["width"]
    new = _lens(case)
    cached = [r.randint(0, case["cached"]) for _ in range(n)]
    held = [-(-c // bs) for c in cached]
    want = sum(max(0, -(-(c + x) // bs) - h) for c, x, h in zip(cached, new, held))
    ids = list(range(sum(held) + want + 1000))  # a pool that others hold parts of
    random.Random(seed).shuffle(ids)
    tables = torch.zeros((n, w), dtype=torch.int32)
    at = 0
    for b, h in enumerate(held):
        tables[b, :h] = torch.tensor(ids[at:at + h], dtype=torch.int32)
        at += h
    free = torch.tensor(ids[at:at + want + 5], dtype=torch.int32, device="cuda")
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return dict(new=dev(new), cached=dev(cached), tables=tables.cuda(), free=free, block=bs,
                tokens=sum(new) + case["slack"])


def _run_maps(s):
    if own:
        from awesome_acceleration_amd import paged
        m = paged.build_step_maps(s["new"], s["cached"], s["tables"], s["block"], s["tokens"],
                                  free_blocks=s["free"])
        return {"tables": s["tables"], "cu": m.cu_seqlens, "positions": m.positions,
                "slots": m.slot_mapping, "ctx": m.context_lens, "taken": m.blocks_taken}
    new, cached, tables, bs = s["new"], s["cached"], s["tables"], s["block"]
    n, w = tables.shape
    ctx = new + cached
    held = ((cached + bs - 1) // bs).clamp(max=w)
    want = ((ctx + bs - 1) // bs).clamp(max=w) - held
    cum = torch.cumsum(want, 0, dtype=torch.int32)
    j = torch.arange(w, device="cuda", dtype=torch.int32)[None]
    at = (cum - want)[:, None] + j - held[:, None]
    fresh = (j >= held[:, None]) & (j < (held + want)[:, None])
    from_free = torch.where(at < s["free"].numel(), s["free"][at.clamp(0, s["free"].numel() - 1)], -1)
    tables.copy_(torch.where(fresh, from_free, tables))
    cu = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    cu[1:] = torch.cumsum(new, 0)
    i = torch.arange(s["tokens"], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(cu[1:], i, right=True).clamp(max=n - 1)
    inside = i < cu[-1]
    pos = torch.where(inside, cached[b] + i - cu[b], 0).long()
    blk = tables[b, (pos // bs).clamp(max=w - 1)].long()
    slots = torch.where(inside & (pos // bs < w) & (blk >= 0), blk * bs + pos % bs, -1)
    return {"tables": tables, "cu": cu, "positions": pos, "slots": slots, "ctx": ctx,
            "taken": cum[-1:]}


# ------------------------------------------------------------------ log probabilities
def _prepare_logprobs(case, seed):
    g, r, c = _gen(seed), case["rows"], case["cols"]
    x = torch.empty((r, c), dtype=DTYPES[case["dtype"]], device="cuda")
    for part in x.split(512):
        y = _randn(g, part.shape[0], c) * 2.5
        # a trained model's rows have a few likely tokens
        at = torch.randint(0, c, (part.shape[0], 1), generator=g, device="cuda")
        at = (at + torch.arange(8, device="cuda") * (c // 8)) % c
        y.scatter_(1, at, 6.0 + 4.0 * _randn(g, part.shape[0], 8))
        if case["allowed"]:  # a grammar leaves some tokens
            keep = torch.zeros(part.shape[0], c, dtype=torch.bool, device="cuda")
            keep.scatter_(1, torch.randint(0, c, (part.shape[0], case["allowed"]), generator=g,
                                           device="cuda"), True)
            y.masked_fill_(~keep, -math.inf)
        part.copy_(y)
    if case["allowed"]:
        tokens = x.argmax(-1)
    else:
        tokens = torch.randint(0, c, (r,), generator=g, device="cuda")
    return dict(x=x, tokens=tokens, top=case["top"])


def _run_logprobs(s):
    if own:
        from awesome_acceleration_amd import fused
        m = fused.token_logprobs(s["x"], s["tokens"], s["top"])
        return {"logprobs": m.logprobs, "entropy": m.entropy, "top": m.top_logprobs, "ids": m.top_ids}
    out = []
    for x, t in zip(s["x"].split(256), s["tokens"].split(256)):
        x = x.float()
        d = x - x.amax(-1, keepdim=True)
        e = torch.exp(d)
        total = e.sum(-1, keepdim=True)
        log = torch.log(total)
        entropy = log[:, 0] - torch.where(e > 0, e * d, 0.0).sum(-1) / total[:, 0]
        ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :s["top"]]
        out.append((d.gather(1, t[:, None])[:, 0] - log[:, 0], entropy, d.gather(1, ids) - log, ids))
    return {k: torch.cat(v) for k, v in zip(("logprobs", "entropy", "top", "ids"), zip(*out))}


def _exact_logprobs(case, seed):
    s = _prepare_logprobs(case, seed)
    got = {k: [] for k in ("logprobs", "entropy", "top", "ids")}
    for x, t in zip(s["x"].split(256), s["tokens"].split(256)):
        lp = torch.log_softmax(x.double(), -1)
        got["logprobs"].append(lp.gather(1, t[:, None])[:, 0])
        got["entropy"].append(-torch.nan_to_num(lp.exp() * lp, nan=0.0).sum(-1))
        # order by (value, lowest index): one whole number for both
        bits = x.float().view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20)
        key = key - torch.arange(x.shape[1], device="cuda")
        ids = torch.topk(key, s["top"], -1)[1]
        got["top"].append(lp.gather(1, ids))
        got["ids"].append(ids)
    return {k: torch.cat(v) for k, v in got.items()}


# ------------------------------------------------------------------ the interface
_PREPARE = dict(store=_prepare_store, attend=_prepare_attend, append=_prepare_attend,
                maps=_prepare_maps, logprobs=_prepare_logprobs)
_RUN = dict(store=_run_store, attend=_run_attend, append=_run_append, maps=_run_maps,
            logprobs=_run_logprobs)


def prepare(case, seed):
    s = _PREPARE[case["kind"]](case, seed)
    s["kind"] = case["kind"]
    return s


def run(state):
    return _RUN[state["kind"]](state)


def exact(case, seed):
    kind = case["kind"]
    if kind == "store":
        return _exact_store(case, seed)
    if kind in ("attend", "append"):
        return _exact_attend(case, seed)
    if kind == "logprobs":
        return _exact_logprobs(case, seed)
    return None  # whole numbers


def work(case):
    kind = case["kind"]
    if kind == "store":
        n = case["tokens"] * case["hkv"]
        es = DTYPES[case["dtype"]].itemsize
        # rows in, 4-bit rows out; 4-bit rows in, rows out
        return {"bytes": 2 * n * (2 * D * es + 136) + 16 * case["tokens"], "flops": 4 * n * 2 * D}
    if kind in ("attend", "append"):
        tokens, es = sum(_lens(case)), DTYPES[case["dtype"]].itemsize
        rows = case["seqs"] * case["hq"] * D * es * 2
        if kind == "append":
            rows += case["seqs"] * case["hkv"] * (2 * 2 * D * es + 2 * 136)
        return {"bytes": tokens * case["hkv"] * 136 + rows + 4 * (tokens // case["block"]),
                "flops": 4 * tokens * case["hq"] * D}
    if kind == "maps":
        tokens = sum(_lens(case)) + case["slack"]
        return {"bytes": 16 * tokens + 16 * case["seqs"] + 4 * case["seqs"] * case["width"],
                "flops": 8 * tokens}
    n = case["rows"] * case["cols"]
    return {"bytes": n * DTYPES[case["dtype"]].itemsize + case["rows"] * (16 + 12 * case["top"]),
            "flops": 5 * n}
