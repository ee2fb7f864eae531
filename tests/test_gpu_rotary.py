"""Rotary positions on the GPU against a plain float64 computation: the rotation, the append
with the rotation on the way, the tables."""
import math

import pytest
import torch

from awesome_acceleration_amd import rotary

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _say(*a):
    print("case:", *a, flush=True)


def _turn(x, cos, sin, inter):
    """float64; x [..., H, D], cos and sin [..., R / 2] of its tokens."""
    h = cos.shape[-1]
    x = x.double().clone()
    c, s = cos.double().unsqueeze(-2), sin.double().unsqueeze(-2)
    a, b = (x[..., :2 * h:2], x[..., 1:2 * h:2]) if inter else (x[..., :h], x[..., h:2 * h])
    y0, y1 = a * c - b * s, a * s + b * c
    if inter:
        x[..., :2 * h:2], x[..., 1:2 * h:2] = y0, y1
    else:
        x[..., :h], x[..., h:2 * h] = y0.clone(), y1
    return x


def _size(x, cos, sin, inter):
    """|x1 c| + |x2 s| of every element, and of the dims that pass: 0."""
    h = cos.shape[-1]
    y = _turn(x.abs(), cos.abs(), -sin.abs(), inter)         # x1 c + x2 s
    z = _turn(x.abs(), cos.abs(), sin.abs(), inter)          # x1 s + x2 c in the second dims
    out = torch.zeros_like(y)
    first = torch.zeros(x.shape[-1], dtype=torch.bool, device=x.device)
    first[0:2 * h:2] = True if inter else first[0:2 * h:2]
    if not inter:
        first[:h] = True
    second = torch.zeros_like(first)
    second[:2 * h] = ~first[:2 * h]
    out[..., first], out[..., second] = y[..., first], z[..., second]
    return out


def _check(got, x, cos, sin, inter):
    """Two float products and a sum (2^-24 of each term twice), one rounding to the type; fp16
    results below 2^-14 are 2^-25 off at most."""
    ref, size = _turn(x, cos, sin, inter), _size(x, cos, sin, inter)
    u = torch.finfo(got.dtype).eps / 2
    lim = u * ref.abs() + (1 + u) * 2.0 ** -23 * size + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    bad = (got.double() - ref).abs() > lim
    assert not bad.any(), f"{int(bad.sum())} beyond the bound"
    keep = 2 * cos.shape[-1]
    assert torch.equal(got[..., keep:], x[..., keep:])


def _tab(gpu, n, rot, dt, seed=0):
    a = torch.rand(n, rot // 2, generator=torch.Generator(device=gpu).manual_seed(seed), device=gpu) * 6.3
    return a.cos().to(dt), a.sin().to(dt)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("table", ["same", "fp32"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, S, H, D, rot", [
    (1, 1, 1, 128, 128), (3, 7, 5, 128, 64), (2, 33, 24, 64, 64), (1, 40, 3, 256, 32), (2, 5, 4, 96, 96),
    (2, 5, 3, 20, 6), (1, 3, 2, 128, 120), (2, 300, 16, 128, 128), (1, 9, 2, 1024, 16), (1, 9, 2, 2, 2)])
def test_rotation(gpu, B, S, H, D, rot, dtype, table, inter):
    _say("rotate", B, S, H, D, rot, dtype, table, inter)
    dt = DTYPES[dtype]
    x = torch.randn(B, S, H, D, device=gpu, generator=torch.Generator(device=gpu).manual_seed(S)).to(dt)
    cos, sin = _tab(gpu, S + 60, rot, dt if table == "same" else torch.float32)
    for off in (7, torch.arange(B, dtype=torch.int32, device=gpu) * 29):
        at = torch.arange(S, device=gpu) + (off if isinstance(off, int) else off.long()[:, None])
        c, s = (t[at.expand(B, S)] for t in (cos, sin))
        got = rotary.apply_rotary_emb(x, cos, sin, inter, seqlen_offsets=off)
        _check(got, x, c, s, inter)
        back = rotary.apply_rotary_emb(x, cos, sin, inter, seqlen_offsets=off, conjugate=True)
        _check(back, x, c, -s, inter)
        y = x.clone()
        assert rotary.apply_rotary_emb(y, cos, sin, inter, inplace=True, seqlen_offsets=off) is y
        assert torch.equal(y, got)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rotation_of_strided_and_misaligned_heads(gpu, dtype):
    _say("strides", dtype)
    dt = DTYPES[dtype]
    cos, sin = _tab(gpu, 50, 64, torch.float32)
    base = torch.randn(3, 50, 12, 128, device=gpu).to(dt)
    flat = torch.randn(3 * 50 * 12 * 128 + 1, device=gpu).to(dt)
    views = [base[:, :, 2:7], base.transpose(1, 2)[:, :, :5].transpose(1, 2), base[:, ::2, ::3],
             base.transpose(0, 1)[:3, :, :4], flat[1:].view(3, 50, 12, 128), base[..., 3:3 + 100],
             base[:1].expand(3, -1, -1, -1)]
    for x in views:
        B, S = x.shape[:2]
        got = rotary.apply_rotary_emb(x, cos, sin, seqlen_offsets=0)
        _check(got, x, cos[:S].expand(B, S, -1), sin[:S].expand(B, S, -1), False)
        keep = base.clone()
        if x.data_ptr() >= base.data_ptr() and x.stride(0):
            y = keep.as_strided(x.shape, x.stride(), x.storage_offset()) if x._base is base else None
            if y is not None:
                rotary.apply_rotary_emb(y, cos, sin, inplace=True)
                assert torch.equal(y, got)
                other = torch.ones_like(keep, dtype=torch.bool)
                other.as_strided(x.shape, x.stride(), x.storage_offset()).fill_(False)
                assert torch.equal(keep[other], base[other])


def test_rotation_of_packed_sequences(gpu):
    _say("packed")
    for lens in ([3, 0, 5, 1], [0, 0, 4], [2] * 70 + [0] * 70 + [3] * 60, [1] * 4200):
        n = sum(lens)
        cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=gpu)
        off = torch.arange(len(lens), dtype=torch.int32, device=gpu) % 40
        x = torch.randn(n + 2, 3, 128, device=gpu).to(torch.bfloat16)
        cos, sin = _tab(gpu, 50, 128, torch.float32)
        at = torch.cat([torch.arange(m) + o for m, o in zip(lens, off.tolist())]).to(gpu)
        y = x.clone()
        rotary.apply_rotary_emb(y, cos, sin, inplace=True, seqlen_offsets=off, cu_seqlens=cu)
        _check(y[:n], x[:n], cos[at], sin[at], False)
        assert torch.equal(y[n:], x[n:])  # rows of no sequence
        got = rotary.apply_rotary_emb(x, cos, sin, seqlen_offsets=off, cu_seqlens=cu)
        assert torch.equal(got[:n], y[:n])


def test_positions_outside_the_tables_take_their_ends(gpu):
    _say("ends")
    x = torch.randn(2, 5, 2, 128, device=gpu)
    cos, sin = _tab(gpu, 4, 128, torch.float32)
    off = torch.tensor([-3, (1 << 31) - 2], dtype=torch.int32, device=gpu)
    at = torch.tensor([[0, 0, 0, 0, 1], [3] * 5], device=gpu)
    _check(rotary.apply_rotary_emb(x, cos, sin, seqlen_offsets=off), x, cos[at], sin[at], False)


def test_special_values_stay_in_their_pair(gpu):
    _say("special")
    x = torch.randn(1, 2, 2, 128, device=gpu)
    x[0, 0, 0, 3], x[0, 1, 1, 70], x[0, 0, 1, 127] = math.inf, math.nan, -math.inf
    cos, sin = _tab(gpu, 4, 96, torch.float32)
    got = rotary.apply_rotary_emb(x, cos, sin)
    ref = _turn(x, cos[:2].expand(1, 2, -1), sin[:2].expand(1, 2, -1), False)
    assert torch.equal(torch.isfinite(got), torch.isfinite(ref)) and got[0, 0, 1, 127] == -math.inf


# ------------------------------------------------------------------ append
def _paged(gpu, ctx, bs, hkv, D, dt, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    need = [max(1, -(-c // bs)) for c in ctx]
    order = torch.randperm(sum(need) + 2, generator=g, device=gpu).to(torch.int32)
    t = torch.zeros((len(ctx), max(need)), dtype=torch.int32, device=gpu)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    kc, vc = (torch.randn((sum(need) + 2, bs, hkv, D), generator=g, device=gpu).to(dt) for _ in "kv")
    return kc, vc, t


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq, hkv, D, rot, bs", [(16, 8, 128, 128, 16), (4, 4, 128, 64, 7), (6, 1, 80, 20, 48),
                                                 (24, 3, 64, 64, 256)])
@pytest.mark.parametrize("packed", [False, True])
def test_append(gpu, hq, hkv, D, rot, bs, dtype, inter, packed):
    _say("append", hq, hkv, D, rot, bs, dtype, inter, packed)
    dt = DTYPES[dtype]
    new = [3, 0, 40, 1] if packed else [6] * 4
    cached = [0, 9, 15, 300]
    n = sum(new)
    x = torch.randn(n, hq + 2 * hkv, D, device=gpu).to(dt)
    q, k, v = x.split((hq, hkv, hkv), 1)
    kc, vc, t = _paged(gpu, [a + b for a, b in zip(new, cached)], bs, hkv, D, dt)
    cos, sin = _tab(gpu, 400, rot, torch.float32)
    pos = torch.cat([torch.arange(m) + c for m, c in zip(new, cached)]).to(gpu)
    seq = torch.cat([torch.full((m,), b) for b, m in enumerate(new)]).to(gpu)
    rows = t[seq, pos // bs].long() * bs + pos % bs
    lens = torch.tensor(cached, dtype=torch.int32, device=gpu)
    before = kc.clone(), vc.clone()
    a = {}
    if packed:
        a["cu_seqlens"] = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=gpu)
    else:
        q, k, v = (i.view(4, 6, -1, D) for i in (q, k, v))
    out = rotary.rotary_append_paged(q, k, v, kc, vc, t, lens, cos, sin, interleaved=inter, **a)
    assert out.shape == q.shape
    q, k, v = (i.reshape(n, -1, D) for i in (q, k, v))
    _check(out.reshape(n, hq, D), q, cos[pos], sin[pos], inter)
    flat = kc.view(-1, hkv, D)
    _check(flat[rows], k, cos[pos], sin[pos], inter)
    assert torch.equal(vc.view(-1, hkv, D)[rows], v)
    rest = torch.ones(flat.shape[0], dtype=torch.bool, device=gpu)
    rest[rows] = False
    for c, w in zip((kc, vc), before):
        assert torch.equal(c.view(-1, hkv, D)[rest], w.view(-1, hkv, D)[rest])
    # without tables and queries: the append alone
    k2 = k if packed else k.view(4, 6, hkv, D)
    v2 = v if packed else v.view(4, 6, hkv, D)
    kc2, vc2 = before[0].clone(), before[1].clone()
    assert rotary.rotary_append_paged(None, k2, v2, kc2, vc2, t, lens, **a) is None
    assert torch.equal(kc2.view(-1, hkv, D)[rows], k) and torch.equal(vc2, vc)
    assert lens.tolist() == cached


def test_append_skips_what_has_no_block(gpu):
    _say("append skips")
    kc = torch.zeros(3, 16, 2, 128, device=gpu, dtype=torch.bfloat16)
    vc = torch.zeros_like(kc)
    t = torch.tensor([[1, -1], [3, 2], [0, 1 << 30], [0, 0]], dtype=torch.int32, device=gpu)
    lens = torch.tensor([14, 14, 30, -2], dtype=torch.int32, device=gpu)
    k = torch.ones(4, 4, 2, 128, device=gpu, dtype=torch.bfloat16)
    q = torch.randn(4, 4, 4, 128, device=gpu).to(torch.bfloat16)
    cos, sin = _tab(gpu, 64, 128, torch.bfloat16)
    out = rotary.rotary_append_paged(q, k, k, kc, vc, t, lens, cos, sin)
    rows = vc[..., 0, 0].nonzero().tolist()
    # sequence 0: 14, 15 in block 1, then none; 1: none, then 0, 1 of block 2; 2: past the
    # table and a bad block; 3: negative lengths store nothing
    assert rows == [[1, 14], [1, 15], [2, 0], [2, 1]]
    at = (torch.arange(4, device=gpu) + lens.long()[:, None]).clamp(0, 63)
    _check(out, q, cos[at], sin[at], False)


def test_append_past_4_gib_and_large(gpu):
    """Rows far into a cache, and enough of them that a wave takes several."""
    _say("append 4 GiB")
    bs, hkv = 256, 8
    nb = (5 << 30) // (bs * hkv * 256)
    kc = torch.empty((nb, bs, hkv, 128), dtype=torch.bfloat16, device=gpu)
    vc = torch.empty_like(kc)
    n = 4000
    t = torch.arange(nb - 1, nb - 1 - 16, -1, dtype=torch.int32, device=gpu).view(1, 16)
    x = torch.randn(1, n, 32, 128, device=gpu).to(torch.bfloat16)
    q, k, v = x.split((16, 8, 8), 2)
    cos, sin = _tab(gpu, n + 50, 128, torch.float32)
    lens = torch.tensor([50], dtype=torch.int32, device=gpu)
    out = rotary.rotary_append_paged(q, k, v, kc, vc, t, lens, cos, sin)
    pos = torch.arange(n, device=gpu) + 50
    blk = t[0, pos // bs].long()
    _check(out[0], q[0], cos[pos], sin[pos], False)
    _check(kc[blk, pos % bs], k[0], cos[pos], sin[pos], False)
    assert torch.equal(vc[blk, pos % bs], v[0])


# ------------------------------------------------------------------ tables
@pytest.mark.parametrize("scaling", [
    None, dict(rope_type="default"), dict(type="linear", factor=3.0),
    dict(rope_type="dynamic", factor=2.0, original_max_position_embeddings=100),
    dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768),
    dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
         original_max_position_embeddings=8192)], ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_tables(gpu, dtype, scaling):
    """The float angle of the reduced position is off by 2^-24 of it at most (an eighth of a
    turn, 0.79), float sine, cosine and factor by 4 units of 2^-24, the result by half a
    step of its type (fp16 below 2^-14: 2^-25)."""
    _say("tables", dtype, scaling)
    dt = DTYPES[dtype]
    for rot, start, n in ((128, 0, 300), (6, 999000, 77), (64, (1 << 31) - 5, 40), (32, -20, 33)):
        r = rotary.RotaryEmbedding(rot, 10000.0, scaling, seq_len=5000, device=gpu)
        # in long doubles' place: the angle modulo 2 pi from its whole and fractional turns
        p = torch.arange(start, start + n, dtype=torch.float64)
        turns = p[:, None] * (r.frequencies / (2 * math.pi))
        turns = turns - turns.round()
        f = float(torch.tensor(r.factor, dtype=torch.float32))
        want = [f * torch.cos(turns * 2 * math.pi), f * torch.sin(turns * 2 * math.pi)]
        u = torch.finfo(dt).eps / 2
        got = r.cos_sin(n, start=start, dtype=dt)
        # (the turns here and there: a product's rounding in 64 bits, 2^-53 of the turns)
        err = float(p.abs().max()) * 2.0 ** -50
        for g, w in zip(got, want):
            lim = u * w.abs() + f * (6 * 2.0 ** -24 + err) + (2.0 ** -25 if dt == torch.float16 else 0)
            assert g.dtype == dt and g.shape == (n, rot // 2)
            assert ((g.cpu().double() - w).abs() <= lim).all()
        if abs(start) < 1 << 30:
            at = torch.arange(start, start + n, dtype=torch.int32, device=gpu).flip(0)
            for g, h in zip(got, r.cos_sin(positions=at, dtype=dt)):
                assert torch.equal(g.flip(0), h)
    assert r.cos_sin(0)[0].shape == (0, 16)


def test_refusals(gpu):
    x = torch.zeros(2, 3, 4, 128, device=gpu, dtype=torch.bfloat16)
    cos, sin = _tab(gpu, 9, 64, torch.float32)
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)  # noqa: E731

    def no(match, f, *a, **o):
        with pytest.raises(RuntimeError, match=match):
            f(*a, **o)

    r = rotary.apply_rotary_emb
    no("GPU", r, x.cpu(), cos, sin)
    no("x must be", r, x[0], cos, sin)
    no("x must be", r, x, cos, sin, cu_seqlens=i(2))
    no("even", r, x[..., :7], cos[:, :3], sin[:, :3])
    no("cos and sin must be contiguous", r, x, cos[:, ::2], sin[:, ::2])
    no("cos and sin must be contiguous", r, x, cos, sin[:5])
    no("heads' dtype", r, x, cos.half(), sin.half())
    no("heads' dtype", r, x, cos, sin.to(torch.bfloat16))
    no("larger than", r, x[..., :32], cos, sin)
    no("empty", r, x, cos[:0], sin[:0])
    no("unsupported dtype", r, x.double(), cos.double(), sin.double())
    no("head_dim must be contiguous", r, x.transpose(2, 3), cos[:, :1].contiguous(), sin[:, :1].contiguous())
    no("seqlen_offsets", r, x, cos, sin, seqlen_offsets=i(3))
    no("seqlen_offsets", r, x, cos, sin, seqlen_offsets=i(2).long())
    no("32 bits", r, x, cos, sin, seqlen_offsets=1 << 31)
    no("broadcast", r, x[:, :1].expand(2, 3, 4, 128), cos, sin, inplace=True)
    no("cu_seqlens", r, x[0], cos, sin, cu_seqlens=i(2).long())
    kc = torch.zeros(5, 16, 4, 128, device=gpu, dtype=torch.bfloat16)
    a = rotary.rotary_append_paged
    t, n = i(2, 3), i(2)
    no("go together", a, x, x, x, kc, kc, t, n, cos)
    no("caches", a, x, x, x, kc, kc[:3], t, n)
    no("caches", a, x, x, x, kc.transpose(0, 1), kc.transpose(0, 1), t, n)
    no("k and v", a, x, x, x[:, :2], kc, kc, t, n)
    no("k and v", a, x, x[:, :, :2], x[:, :, :2], kc, kc, t, n)
    no("mismatch", a, x, x.half(), x.half(), kc, kc, t, n)
    no("q must be", a, x[:, :2], x, x, kc, kc, t, n)
    no("q must be", a, x.half(), x, x, kc, kc, t, n)
    no("cache_seqlens", a, x, x, x, kc, kc, t, i(3))
    no("cache_seqlens", a, x, x, x, kc, kc, t, n.long())
    no("block_tables", a, x, x, x, kc, kc, t.long(), n)
    no("block_tables", a, x, x, x, kc, kc, i(3, 3), n)
    no("block_tables", a, x, x, x, kc, kc, i(2, 0), n)
    e = rotary.RotaryEmbedding(64, device=gpu)
    no("n must", e.cos_sin)
    no("positions, or", e.cos_sin, 5, positions=i(5))
    no("positions must", e.cos_sin, positions=i(5).long())
    no("unsupported dtype", e.cos_sin, 5, dtype=torch.float64)
    no("inconsistent", e.cos_sin, 5, start=1 << 50)


def test_a_cache_without_blocks_is_refused(gpu):
    q = torch.zeros(2, 3, 4, 128, device=gpu, dtype=torch.bfloat16)
    cache = torch.zeros(0, 16, 4, 128, device=gpu, dtype=torch.bfloat16)
    cos, sin = _tab(gpu, 9, 64, torch.float32)
    with pytest.raises(RuntimeError, match="not empty"):
        rotary.rotary_append_paged(q, q, q, cache, cache, torch.zeros(2, 1, dtype=torch.int32, device=gpu),
                                   torch.zeros(2, dtype=torch.int32, device=gpu), cos, sin)


def test_as_many_tokens_as_a_launch_takes(gpu):
    """2^26 - 4 heads of two dims; one token more is refused."""
    _say("2^26 tokens")
    n = (1 << 26) - 4
    x = torch.randn((1, n + 1, 1, 2), device=gpu, dtype=torch.bfloat16)
    cos, sin = _tab(gpu, 1000, 2, torch.float32)
    got = rotary.apply_rotary_emb(x[:, :n], cos, sin)
    for a in (0, n // 2, n - 1500):
        at = torch.arange(a, a + 1500, device=gpu).clamp(max=999)
        _check(got[0, a:a + 1500], x[0, a:a + 1500], cos[at], sin[at], False)
    with pytest.raises(RuntimeError, match="unsupported"):
        rotary.apply_rotary_emb(x, cos, sin)


def test_no_start_is_cut_to_64_bits(gpu):
    e = rotary.RotaryEmbedding(64, device=gpu)
    for start in ((1 << 64) + 5, -(1 << 64), 1 << 63, (1 << 40) + 1, -(1 << 40) - 1):
        with pytest.raises(RuntimeError, match="inconsistent"):
            e.cos_sin(5, start=start)
    for start in (1 << 40, -(1 << 40)):
        assert e.cos_sin(5, start=start)[0].shape == (5, 32)
