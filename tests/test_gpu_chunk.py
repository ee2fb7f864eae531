"""Chunks of new tokens over the paged cache on the GPU (prefill_paged, flash_attn_varlen_func
with a block table, flash_attn_with_kvcache of several tokens) against a plain float64
computation."""
import math

import pytest
import torch

from awesome_acceleration_amd import flash_attn_interface as fai
from awesome_acceleration_amd import rotary

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
SCALE = 128 ** -0.5


def _say(*a):
    print("case:", *a, flush=True)


def _gen(gpu, seed):
    return torch.Generator(device=gpu).manual_seed(seed)


def _make(gpu, seed, new, ctx, hq, hkv, bs, dt, spare=3, extra_rows=0):
    """Queries, caches filled everywhere, shuffled tables, cu_seqlens, context lengths."""
    g = _gen(gpu, seed)
    need = [max(1, -(-c // bs)) for c in ctx]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=g, device=gpu).to(torch.int32)
    tables = torch.full((len(ctx), max(need) + 1), -7, dtype=torch.int32, device=gpu)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    rnd = lambda *s: torch.randn(s, generator=g, device=gpu).to(dt)  # noqa: E731
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=gpu)
    return dict(q=rnd(sum(new) + extra_rows, hq, 128), kc=rnd(pool, bs, hkv, 128) * 1.5,
                vc=rnd(pool, bs, hkv, 128), tables=tables, cu=cu, new=new, lens=ctx,
                ctx=torch.tensor(ctx, dtype=torch.int32, device=gpu), bs=bs)


def _rows(x, cache, b, n):
    at = torch.arange(n, device=cache.device)
    blk = x["tables"][b].long()[at // x["bs"]]
    blk = torch.where((blk >= 0) & (blk < cache.shape[0]), blk, 0)
    return cache[blk, at % x["bs"]].double()


def _reference(x, causal, scale=SCALE):
    """(out, sum p |v|, the largest sum |q||k| scale of a row) in float64; what a query does
    not see takes no part."""
    q = x["q"].double()
    hq, hkv = q.shape[1], x["kc"].shape[2]
    g = hq // hkv
    out = torch.zeros_like(q)
    absv, z = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    a = 0
    for b, (n, L) in enumerate(zip(x["new"], x["lens"])):
        if n and L:
            k, v = _rows(x, x["kc"], b, L), _rows(x, x["vc"], b, L)
            i = torch.arange(n, device=q.device)[:, None]
            hide = torch.arange(L, device=q.device)[None] > (i + L - n if causal else i + L)
            for h in range(hq):
                qq, kk, vv = q[a:a + n, h], k[:, h // g].contiguous(), v[:, h // g].contiguous()
                s = (qq @ kk.t().contiguous() * scale).masked_fill(hide, -math.inf)
                p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
                p = torch.where(hide.all(-1, keepdim=True), torch.zeros_like(p), p)
                out[a:a + n, h] = p @ vv
                absv[a:a + n, h] = p @ vv.abs()
                z[a:a + n, h] = (qq.abs() @ kk.abs().t().contiguous() * scale).amax(-1)
        a += n
    return out, absv, z


def _check(got, x, causal, scale=SCALE, what=""):
    """With A = sum p |v|, u half a step of the type (bf16 2^-8, fp16 2^-11) and z the largest
    sum |q||k| scale of the row: the probabilities are rounded above and below the fraction
    line (2 u A), the result once (u |out|); a score is a float sum of 128 products whose
    error moves its probability by 2^-17 z at most, and sums and exponentials in float, some
    thousand terms, by 2^-15.  fp16 probabilities below 2^-14 (of a largest of 1 or more) are
    2^-25 off at most, and so are results there."""
    ref, absv, z = _reference(x, causal, scale)
    n = sum(x["new"])
    o = got[:n].double()
    assert torch.isfinite(o).all(), what
    u = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -11
    lim = u * ref[:n].abs() + (2 * u + 2.0 ** -15 + 2.0 ** -16 * z[:n, :, None]) * absv[:n]
    if got.dtype == torch.float16:
        lim = lim + 2.0 ** -25 * (1 + max(x["lens"]) * float(x["vc"].double().abs().nan_to_num(0, 0, 0).max()))
    bad = (o - ref[:n]).abs() > lim
    assert not bad.any(), f"{what}: {int(bad.sum())} beyond the bound, worst {float(((o - ref[:n]).abs() - lim).max()):.3e}"


def _run(x, causal, **o):
    return fai.prefill_paged(x["q"], x["kc"], x["vc"], x["cu"], x["tables"], x["ctx"],
                             max(x["new"], default=0), causal=causal, **o)


CASES = [
    # (new, context), heads, block
    ("one token", [1], [1], 16, 8, 16),
    ("a chunk alone", [5], [5], 16, 8, 16),
    ("draft tokens", [5] * 4, [1031, 17, 255, 256], 16, 8, 256),
    ("ragged", [0, 1, 33, 64, 100, 0, 7], [9, 1, 33, 65, 300, 0, 2000], 16, 8, 16),
    ("odd pages", [3, 40], [50, 101], 8, 4, 48),
    ("pages of a token", [2, 19], [5, 40], 4, 2, 1),
    ("pages of seven", [2, 70], [50, 200], 8, 2, 7),
    ("one head a group", [130, 3], [400, 3], 4, 4, 64),
    ("group of four", [17, 40, 33], [600, 64, 33], 32, 8, 64),
    ("group of eight", [17, 4], [300, 90], 16, 2, 32),
    ("group of three", [50, 4], [300, 90], 6, 2, 32),
    ("group of twelve", [30, 9], [210, 90], 12, 1, 32),
    ("more queries than keys", [40, 9], [7, 0], 16, 8, 16),
    ("several row blocks", [300, 257], [900, 1300], 16, 8, 64),
    ("split keys", [40], [9000], 8, 1, 64),
    ("split keys, few rows", [2, 3], [20000, 700], 4, 1, 256),
    ("split keys, many rows", [513], [6000], 2, 1, 128),
    # the work of a head shared out over its workgroups, whatever the sequences are
    ("shared, uneven", [300, 1, 0, 77, 130, 2, 260, 0, 19], [4000, 3000, 700, 77, 2500, 0, 3333, 5, 40], 16, 8, 64),
    ("shared, few rows", [1, 3, 0, 7, 2] * 9, [i * 37 % 2600 for i in range(45)], 4, 2, 16),
    ("shared, middle rows", [20, 31, 5, 32], [900, 2000, 1300, 32], 8, 4, 48),
    ("shared, half the rows", [60, 13, 64], [3000, 2000, 1700], 4, 2, 256),
    ("shared, group of three", [100, 40, 7], [1500, 2100, 900], 6, 2, 16),
    ("shared, odd pages", [150, 2, 33], [1000, 1200, 900], 2, 1, 20),
    ("shared, prompts alone", [700, 1, 1300, 90], [700, 1, 1300, 90], 4, 2, 64),
    ("shared, hundreds of sequences", [i % 4 for i in range(300)], [i * 53 % 1500 for i in range(300)], 2, 1, 16),
    ("more sequences than shares take", [i % 2 for i in range(1100)], [i * 7 % 1200 for i in range(1100)], 1, 1, 16),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES, ids=[c[0] for c in CASES])
def test_against_float64(gpu, case, dtype, causal):
    name, new, ctx, hq, hkv, bs = case
    _say(name, dtype, causal)
    x = _make(gpu, len(name), new, ctx, hq, hkv, bs, DTYPES[dtype])
    got = _run(x, causal)
    _check(got, x, causal, what=name)
    again = _run(x, causal, max_context_len=max(max(ctx), 1))
    _check(again, x, causal, what=name + ", with the longest context")
    assert torch.equal(_run(x, causal), got)  # and the same on every run


@pytest.mark.parametrize("new, ctx, hq, hkv, bs", [
    ([9, 1, 4], [500, 40, 2100], 71, 1, 16),    # groups past a wave's rows
    ([3, 2], [700, 300], 600, 2, 64),           # and past a workgroup's
    ([1, 13, 2], [64, 63, 2], 16, 8, 16),       # one iteration of keys at most
    ([64] * 9, [64] * 9, 8, 4, 32),
    ([5, 64], [65, 64], 16, 8, 48),             # and one key more
])
def test_wide_groups_and_short_contexts(gpu, new, ctx, hq, hkv, bs):
    _say("groups", hq, hkv, ctx)
    x = _make(gpu, hq, new, ctx, hq, hkv, bs, torch.bfloat16)
    for causal in (True, False):
        got = _run(x, causal)
        _check(got, x, causal)
        _check(_run(x, causal, max_context_len=max(ctx)), x, causal, what="with the longest context")


def test_slot_layout_of_any_length(gpu):
    """One block a sequence, its length no multiple of anything."""
    _say("slots")
    x = _make(gpu, 4, [7, 40], [333, 70], 16, 8, 335, torch.bfloat16)
    x["tables"] = x["tables"][:, :1].contiguous()
    _check(_run(x, True), x, True)


def test_strides_out_and_rows_behind(gpu):
    _say("strides")
    x = _make(gpu, 5, [9, 40], [100, 41], 16, 8, 16, torch.bfloat16, extra_rows=6)
    wide = torch.zeros(55, 32, 128, dtype=torch.bfloat16, device=gpu)
    wide[:, 8:24] = x["q"]
    x["q"] = wide[:, 8:24]
    out = torch.full((55, 20, 128), 3.0, dtype=torch.bfloat16, device=gpu)
    got = _run(x, True, out=out[:, 4:])
    assert got.data_ptr() == out[:, 4:].data_ptr()
    _check(out[:, 4:], x, True)
    assert (out[:, :4] == 3).all() and (out[49:] == 3).all()


@pytest.mark.parametrize("bs", [16, 7, 256])
@pytest.mark.parametrize("rows", [5, 200])
def test_what_is_not_seen_does_not_matter(gpu, bs, rows):
    """Rows behind the context, keys of later tokens and blocks of no table hold infinities
    and NaN."""
    _say("unseen", bs, rows)
    for dt in DTYPES.values():
        ctx = [rows + 37, rows + 3]
        x = _make(gpu, 6, [rows, rows], ctx, 16, 8, bs, dt)
        used = torch.zeros(x["kc"].shape[:2], dtype=torch.bool, device=gpu)
        for b, n in enumerate(ctx):
            at = torch.arange(n, device=gpu)
            used[x["tables"][b].long()[at // bs], at % bs] = True
        for c in (x["kc"], x["vc"]):
            c[~used] = math.nan
            c[~used, 0, 5] = math.inf
        x["tables"][:, -1] = 1 << 30
        _check(_run(x, True), x, True)
        # the last token's key and value are bad: every query but the last is as before
        at = ctx[0] - 1
        blk = int(x["tables"][0, at // bs])
        want = _run(x, True)
        x["kc"][blk, at % bs, 3, 7] = math.nan
        x["vc"][blk, at % bs, 2, 9] = -math.inf
        x["vc"][blk, at % bs, 5] = math.nan
        got = _run(x, True)
        bad = got != want
        assert not bad[:rows - 1].any() and not bad[rows:].any()
        last = got[rows - 1]
        assert last[4:6, 9].eq(-math.inf).all() and torch.isfinite(last[4:6, :9]).all()
        assert last[10:12].isnan().all() and last[6:8].isnan().all()
        assert torch.isfinite(last[:4]).all() and torch.isfinite(last[12:]).all()


def test_block_numbers_outside_the_cache_are_read_as_block_0(gpu):
    _say("bad blocks")
    x = _make(gpu, 7, [9, 70], [40, 100], 8, 4, 16, torch.bfloat16)
    x["tables"][0, 1] = -3
    x["tables"][1, 2] = x["kc"].shape[0]
    x["tables"][1, 4] = 1 << 30
    _check(_run(x, True), x, True)  # (the reference reads block 0 for them too)


def test_a_context_past_the_table_is_cut_to_it(gpu):
    _say("long context")
    x = _make(gpu, 8, [9], [64], 8, 4, 16, torch.bfloat16)
    x["tables"] = x["tables"][:, :4].contiguous()
    x["ctx"] += 1000
    _check(_run(x, False), x, False)
    x["ctx"].fill_((1 << 31) - 1)
    _check(_run(x, True), x, True)
    # and one whose tokens are appended past its table: none is stored
    lens = torch.tensor([(1 << 31) - 3], dtype=torch.int32, device=gpu)
    k = torch.ones(1, 9, 4, 128, dtype=torch.bfloat16, device=gpu)
    before = x["kc"].clone()
    got = fai.flash_attn_with_kvcache(x["q"].view(1, 9, 8, 128), x["kc"], x["vc"], k=k, v=k, cache_seqlens=lens,
                                      block_table=x["tables"], causal=False)
    assert torch.equal(x["kc"], before)
    _check(got[0], x, False)


def test_more_queries_than_said(gpu):
    """A max_seqlen_q below a sequence's length leaves rows unwritten and reads nothing wrong."""
    _say("understated")
    x = _make(gpu, 9, [300, 5], [300, 50], 16, 8, 16, torch.bfloat16)
    out = torch.full_like(x["q"], 7.0)
    fai.prefill_paged(x["q"], x["kc"], x["vc"], x["cu"], x["tables"], x["ctx"], 128, out=out)
    want = _run(x, True)
    done = (out != 7).flatten(1).all(1)
    assert done[300:].all() and torch.equal(out[done], want[done]) and int(done[:300].sum()) >= 128


def test_caches_past_4_gib(gpu):
    _say("4 GiB")
    bs, hkv = 256, 8
    nb = (5 << 30) // (bs * hkv * 256)
    kc = torch.empty((nb, bs, hkv, 128), dtype=torch.bfloat16, device=gpu)
    vc = torch.empty_like(kc)
    x = _make(gpu, 10, [40, 3], [500, 400], 16, hkv, bs, torch.bfloat16, spare=0)
    small = x["kc"].shape[0]
    x["tables"][x["tables"] >= 0] += nb - small
    kc[nb - small:], vc[nb - small:] = x["kc"], x["vc"]
    x["kc"], x["vc"] = kc, vc
    got = _run(x, True)
    y = dict(x, kc=kc[nb - small:].clone(), vc=vc[nb - small:].clone())
    y["tables"] = torch.where(x["tables"] >= 0, x["tables"] - (nb - small), x["tables"])
    _check(got, y, True)


def test_large_scores_and_the_lowest_values(gpu):
    """Scores whose exponentials overflow without the running maximum, falling and rising."""
    _say("large scores")
    x = _make(gpu, 11, [40], [300], 8, 4, 16, torch.bfloat16)
    x["kc"] *= torch.linspace(-30, 30, x["kc"].shape[0], device=gpu).view(-1, 1, 1, 1).to(torch.bfloat16)
    for causal in (True, False):
        _check(_run(x, causal), x, causal)
    _check(_run(x, True, softmax_scale=1e-3), x, True, scale=1e-3)


def test_varlen_call_with_a_block_table(gpu):
    _say("varlen")
    x = _make(gpu, 12, [9, 0, 130], [100, 3, 131], 16, 8, 64, torch.float16)
    cu_k = torch.cat((torch.zeros(1, dtype=torch.int32, device=gpu), x["ctx"].cumsum(0, dtype=torch.int32)))
    got = fai.flash_attn_varlen_func(x["q"], x["kc"], x["vc"], x["cu"], cu_k, 130, 131, causal=True,
                                     block_table=x["tables"])
    assert torch.equal(got, _run(x, True))


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("sq, sk", [(5, 5), (1, 4), (6, 2), (3, 0), (70, 70)])
def test_kvcache_call_of_several_tokens(gpu, sq, sk, causal, paged):
    """Appended rows bit for bit, then attention over cache_seqlens + S_new tokens."""
    _say("kvcache", sq, sk, causal, paged)
    bs = 16 if paged else 200
    cached = [0, 31, 100]
    x = _make(gpu, 13, [sq] * 3, [c + sk for c in cached], 16, 8, bs, torch.bfloat16)
    g = _gen(gpu, 1)
    qkv = torch.randn((3, max(sq, sk), 32, 128), generator=g, device=gpu).to(torch.bfloat16)
    q, k, v = qkv[:, :sq, :16], qkv[:, :sk, 16:24], qkv[:, :sk, 24:]
    x["q"] = q.reshape(-1, 16, 128)
    want = [c.clone() for c in (x["kc"], x["vc"])]
    for b, c in enumerate(cached):
        for i in range(sk):
            p = c + i
            for w, t in zip(want, (k, v)):
                w[int(x["tables"][b, p // bs]), p % bs] = t[b, i]
    lens = torch.tensor(cached, dtype=torch.int32, device=gpu)
    where = dict(block_table=x["tables"]) if paged else dict(cache_batch_idx=x["tables"][:, 0])
    if not paged:
        x["tables"] = x["tables"][:, :1].contiguous()
    got = fai.flash_attn_with_kvcache(q, x["kc"], x["vc"], k=k, v=v, cache_seqlens=lens, causal=causal,
                                      **where)
    assert got.shape == q.shape and lens.tolist() == cached
    assert torch.equal(x["kc"], want[0]) and torch.equal(x["vc"], want[1])
    _check(got.reshape(-1, 16, 128), x, causal)
    if not sk:
        alone = fai.flash_attn_with_kvcache(q, x["kc"], x["vc"], cache_seqlens=lens, causal=causal, **where)
        assert torch.equal(alone, got)


@pytest.mark.parametrize("hq", [16, 24])
@pytest.mark.parametrize("S", [1, 4])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("inter, rot", [(True, 64), (False, 128)])
def test_kvcache_call_with_rotary(gpu, S, causal, inter, rot, hq):
    """The call is apply_rotary_emb of the new rows, the append and the attention."""
    _say("kvcache rotary", S, causal, inter, rot, hq)
    cached = [0, 31, 100]
    x = _make(gpu, 14, [S] * 3, [c + S for c in cached], hq, 8, 16, torch.bfloat16)
    g = _gen(gpu, 2)
    q, k, v = (torch.randn((3, S, h, 128), generator=g, device=gpu).to(torch.bfloat16) for h in (hq, 8, 8))
    cos, sin = rotary.RotaryEmbedding(rot, device=gpu).cos_sin(200)
    lens = torch.tensor(cached, dtype=torch.int32, device=gpu)
    turned = rotary.apply_rotary_emb(k, cos, sin, inter, seqlen_offsets=lens)
    want = x["kc"].clone()
    for b, c in enumerate(cached):
        for i in range(S):
            want[int(x["tables"][b, (c + i) // 16]), (c + i) % 16] = turned[b, i]
    got = fai.flash_attn_with_kvcache(q, x["kc"], x["vc"], k=k, v=v, rotary_cos=cos, rotary_sin=sin,
                                      cache_seqlens=lens, block_table=x["tables"], causal=causal,
                                      rotary_interleaved=inter)
    assert torch.equal(x["kc"], want)
    x["q"] = torch.cat([rotary.apply_rotary_emb(q[:, i:i + 1], cos, sin, inter,
                                                seqlen_offsets=lens + (i if causal else 0))
                        for i in range(S)], 1).reshape(-1, hq, 128)
    _check(got.reshape(-1, hq, 128), x, causal)


def test_fp32_single_token_with_rotary(gpu):
    """The decode kernels take float32, so a single token does here too."""
    _say("fp32 rotary")
    x = _make(gpu, 15, [1, 1], [4, 30], 8, 4, 16, torch.float32)
    g = _gen(gpu, 3)
    q, k, v = (torch.randn((2, 1, h, 128), generator=g, device=gpu) for h in (8, 4, 4))
    cos, sin = rotary.RotaryEmbedding(128, device=gpu).cos_sin(64)
    lens = x["ctx"] - 1
    got = fai.flash_attn_with_kvcache(q, x["kc"], x["vc"], k=k, v=v, rotary_cos=cos, rotary_sin=sin,
                                      cache_seqlens=lens, block_table=x["tables"],
                                      rotary_interleaved=False)
    x["q"] = rotary.apply_rotary_emb(q, cos, sin, seqlen_offsets=lens)[:, 0]
    ref, absv, z = _reference(x, False)
    # float sums: 2^-17 z of each probability, 2^-15 for sums of some tens of terms and exp
    assert ((got[:, 0].double() - ref).abs() <= (2.0 ** -15 + 2.0 ** -16 * z[..., None]) * absv).all()


@pytest.mark.parametrize("ctx", [300, 9000])
def test_captured_and_replayed(gpu, ctx):
    """A captured step, replayed with other lengths between eager work."""
    _say("graph", ctx)
    x = _make(gpu, 16, [4, 4], [ctx, ctx], 4, 1, 16, torch.bfloat16)
    y = _make(gpu, 17, [4, 4], [ctx, ctx], 4, 1, 16, torch.bfloat16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _run(x, True)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for z in (x, y):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _run(z, True)
        graphs.append((graph, out, z))
    for n in (ctx, ctx - 5, 4, ctx // 2):
        for _, _, z in graphs:
            z["lens"] = [n, max(4, n - 1)]
            z["ctx"].copy_(torch.tensor(z["lens"], device=gpu))
        # both at once on two streams: their workspaces are their own
        streams = [torch.cuda.Stream() for _ in graphs]
        for st, (graph, _, _) in zip(streams, graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                graph.replay()
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        for _, out, z in graphs:
            _check(out, z, True, what=f"replay at {n}")


def test_two_streams_and_threads(gpu):
    _say("streams")
    import threading
    xs = [_make(gpu, 20 + i, [3, 2], [9000, 5000 + i], 4, 1, 64, torch.bfloat16) for i in range(2)]
    want = [_run(x, True) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                if not torch.equal(_run(xs[i], True), want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_refusals(gpu):
    x = _make(gpu, 30, [3, 2], [20, 5], 16, 8, 16, torch.bfloat16)
    q, kc, vc, cu, t, ctx = (x[i] for i in ("q", "kc", "vc", "cu", "tables", "ctx"))

    def no(match, f, *a, err=RuntimeError, **o):
        with pytest.raises(err, match=match):
            f(*a, **o)

    p = fai.prefill_paged
    no("GPU", p, q.cpu(), kc, vc, cu, t, ctx, 3)
    no("fp16 and bf16", p, q.float(), kc.float(), vc.float(), cu, t, ctx, 3)
    no("share a dtype", p, q.half(), kc, vc, cu, t, ctx, 3)
    no("head_dim", p, q[..., :64].contiguous(), kc, vc, cu, t, ctx, 3)
    no("multiple", p, q[:, :12], kc, vc, cu, t, ctx, 3)
    no("contiguous", p, q[..., ::2], kc[..., ::2], vc[..., ::2], cu, t, ctx, 3)
    no("caches must be", p, q, kc[0], vc[0], cu, t, ctx, 3)
    no("contiguous", p, q, kc.transpose(0, 1), vc.transpose(0, 1), cu, t, ctx, 3)
    no("cu_seqlens", p, q, kc, vc, cu.long(), t, ctx, 3)
    no("context_lens", p, q, kc, vc, cu, t, ctx.long(), 3)
    no("context_lens", p, q, kc, vc, cu, t, ctx[:1], 3)
    no("block_tables", p, q, kc, vc, cu, t.long(), ctx, 3)
    no("block_tables", p, q, kc, vc, cu, t[:, ::2], ctx, 3)
    no("positive", p, q, kc, vc, cu, t, ctx, 3, softmax_scale=0.0)
    no("positive", p, q, kc, vc, cu, t, ctx, 3, softmax_scale=-1.0)
    no("out must", p, q, kc, vc, cu, t, ctx, 3, out=torch.empty_like(q).half())
    no("aligned", p, torch.empty(5, 17, 128, dtype=q.dtype, device=gpu).view(-1)[4:4 + q.numel()].view(q.shape),
       kc, vc, cu, t, ctx, 3)
    no("invalid", p, q, kc, vc, cu, t, ctx, -1)
    no("cu_seqlens", fai.flash_attn_varlen_func, q, kc, vc, cu, cu[:2], 3, 20, block_table=t)
    f = fai.flash_attn_with_kvcache
    qq = q[:4].view(2, 2, 16, 128)
    kk = torch.zeros(2, 2, 8, 128, dtype=q.dtype, device=gpu)
    a = dict(cache_seqlens=ctx, block_table=t)
    no("fp16 and", f, qq.float(), kc.float(), vc.float(), **a)
    no("together", f, qq, kc, vc, k=kk, **a)
    no("k/v must", f, qq, kc, vc, k=kk[:1], v=kk[:1], **a)
    no("k/v must", f, qq, kc, vc, k=kk[:, :, :4], v=kk[:, :, :4], **a)
    no("mismatch", f, qq, kc, vc, k=kk.half(), v=kk.half(), **a)
    tab = torch.zeros(64, 64, device=gpu)
    no("new keys", f, qq, kc, vc, rotary_cos=tab, rotary_sin=tab, **a)
    no("rotary_dim", f, qq, kc, vc, k=kk, v=kk, rotary_cos=torch.zeros(9, 65, device=gpu),
       rotary_sin=torch.zeros(9, 65, device=gpu), **a)
    no("without", f, qq, kc, vc, k=kk, v=kk, rotary_cos=tab, err=NotImplementedError, **a)
    no("positive", f, qq, kc, vc, softmax_scale=-1.0, **a)
    before = kc.clone()
    no("heads' dtype", f, qq, kc, vc, k=kk, v=kk, rotary_cos=tab.half(), rotary_sin=tab.half(), **a)
    assert torch.equal(kc, before)


def test_nothing_to_do(gpu):
    x = _make(gpu, 31, [3, 2], [20, 5], 16, 8, 16, torch.bfloat16)
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)  # noqa: E731
    assert fai.prefill_paged(x["q"][:0], x["kc"], x["vc"], i(3), x["tables"], x["ctx"], 0).shape == (0, 16, 128)
    assert fai.prefill_paged(x["q"][:0], x["kc"], x["vc"], i(1), i(0, 4), i(0), 0).shape == (0, 16, 128)
    assert (fai.prefill_paged(x["q"], x["kc"][:0], x["vc"][:0], x["cu"], x["tables"], x["ctx"], 3) == 0).all()
    assert (fai.prefill_paged(x["q"], x["kc"], x["vc"], x["cu"], x["tables"], i(2), 3) == 0).all()
    none = fai.flash_attn_with_kvcache(x["q"][:0].view(0, 4, 16, 128), x["kc"], x["vc"], cache_seqlens=i(0),
                                       block_table=i(0, 3))
    assert none.shape == (0, 4, 16, 128)


@pytest.mark.parametrize("rot", [0, 128])
@pytest.mark.parametrize("sq, sk", [(1, 1), (5, 5), (1, 4), (6, 2), (3, 0)])
def test_kvcache_call_on_slots_by_default(gpu, sq, sk, rot):
    """Neither block_table nor cache_batch_idx: row b uses slot b."""
    _say("slots by default", sq, sk, rot)
    cached = [0, 31, 100]
    x = _make(gpu, 18, [sq] * 3, [c + sk for c in cached], 16, 8, 120, torch.bfloat16)
    x["tables"] = torch.arange(3, dtype=torch.int32, device=gpu).view(3, 1)
    g = _gen(gpu, 4)
    q, k, v = (torch.randn((3, s, h, 128), generator=g, device=gpu).to(torch.bfloat16)
               for s, h in ((sq, 16), (sk, 8), (sk, 8)))
    lens = torch.tensor(cached, dtype=torch.int32, device=gpu)
    a = dict(cache_seqlens=lens, causal=True)
    qt, kt = q, k
    if rot:
        a["rotary_cos"], a["rotary_sin"] = rotary.RotaryEmbedding(rot, device=gpu).cos_sin(200)
        qt, kt = (rotary.apply_rotary_emb(t, a["rotary_cos"], a["rotary_sin"], True, seqlen_offsets=lens)
                  for t in (q, k))
    want = [c.clone() for c in (x["kc"], x["vc"])]
    for b, c in enumerate(cached):
        want[0][b, c:c + sk], want[1][b, c:c + sk] = kt[b], v[b]
    kc, vc = x["kc"].clone(), x["vc"].clone()
    got = fai.flash_attn_with_kvcache(q, x["kc"], x["vc"], k=k, v=v, **a)
    assert torch.equal(x["kc"], want[0]) and torch.equal(x["vc"], want[1])
    x["q"] = qt.reshape(-1, 16, 128)
    _check(got.reshape(-1, 16, 128), x, True)
    # and as with the slots named
    named = fai.flash_attn_with_kvcache(q, kc, vc, k=k, v=v, cache_batch_idx=torch.arange(3, device=gpu), **a)
    assert torch.equal(named, got) and torch.equal(kc, x["kc"]) and torch.equal(vc, x["vc"])
    if sk == 0 and not rot:
        assert torch.equal(fai.flash_attn_with_kvcache(q, kc, vc, **a), got)


@pytest.mark.parametrize("S", [1, 3])
def test_a_refused_call_leaves_the_cache(gpu, S):
    """Heads of 64 dims, which the append takes and the attention does not."""
    _say("refused", S)
    kc, vc = (torch.ones(4, 16, 2, 64, dtype=torch.bfloat16, device=gpu) for _ in "kv")
    q, k = (torch.randn(2, S, h, 64, device=gpu).to(torch.bfloat16) for h in (4, 2))
    cos, sin = rotary.RotaryEmbedding(64, device=gpu).cos_sin(40)
    t = torch.arange(4, dtype=torch.int32, device=gpu).view(2, 2)
    with pytest.raises(RuntimeError, match="head_dim"):
        fai.flash_attn_with_kvcache(q, kc, vc, k=k, v=k, rotary_cos=cos, rotary_sin=sin, cache_seqlens=5, block_table=t)
    assert (kc == 1).all() and (vc == 1).all()


def _part(x, got, seqs):
    """The given sequences of a packed problem whose sequences have one length: a problem and its rows."""
    n, at = x["new"][0], torch.tensor(seqs, device=got.device)
    rows = (at[:, None] * n + torch.arange(n, device=got.device)).flatten()
    return dict(x, q=x["q"][rows], tables=x["tables"][at], new=[n] * len(seqs),
                lens=[x["lens"][b] for b in seqs]), got[rows]


def test_any_bound_of_the_queries_will_do(gpu):
    _say("bounds")
    x = _make(gpu, 32, [3, 40, 1], [300, 41, 9], 16, 8, 16, torch.bfloat16)
    for most in (44, 45, 1 << 20, (1 << 31) - 1, 1 << 31, (1 << 32) + 3, 1 << 40):
        _check(fai.prefill_paged(x["q"], x["kc"], x["vc"], x["cu"], x["tables"], x["ctx"], most), x, True, what=str(most))


def test_more_workgroups_than_a_launch_numbers(gpu):
    """1030 sequences said to be of up to 32,768 queries: 8.4 million workgroups of 512 threads."""
    _say("2^23 workgroups")
    n, L, B = 32, 40, 1030
    x = _make(gpu, 33, [n] * B, [L] * B, 64, 1, 16, torch.bfloat16)
    got = fai.prefill_paged(x["q"], x["kc"], x["vc"], x["cu"], x["tables"], x["ctx"], 1 << 15)
    y, rows = _part(x, got, [0, 1, 500, *range(1018, 1030)])
    _check(rows, y, True)
    # both within 3 half steps of 2^-8 (and float's) of the largest |v| from the same values
    assert (got.float() - _run(x, True).float()).abs().max() <= 2 * 3.1 * 2.0 ** -8 * x["vc"].float().abs().max()


def test_more_sequences_than_a_launch_holds(gpu):
    """65,537 sequences of two tokens, 128 KV heads: the same without cu_seqlens."""
    _say("2^23 sequences' heads")
    B, h = 65537, 128
    x = _make(gpu, 34, [2] * 8, [16] * 8, h, h, 16, torch.bfloat16)
    g = _gen(gpu, 5)
    q = torch.randn((B, 2, h, 128), generator=g, device=gpu, dtype=torch.bfloat16)
    lens = torch.randint(1, 17, (B,), generator=g, device=gpu, dtype=torch.int32)
    tables = torch.randint(0, x["kc"].shape[0], (B, 1), generator=g, device=gpu, dtype=torch.int32)
    got = fai.flash_attn_with_kvcache(q, x["kc"], x["vc"], cache_seqlens=lens, block_table=tables, causal=True)
    x.update(q=q.view(-1, h, 128), tables=tables, new=[2] * B, lens=lens.tolist())
    y, rows = _part(x, got.view(-1, h, 128), [0, 40000, 65533, 65534, 65535, 65536])
    _check(rows, y, True)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("none", ["blocks", "columns", "keys"])
def test_rows_of_no_sequence_without_any_key(gpu, none):
    """Zeros for the sequences' rows; those before and behind them stay."""
    _say("no key", none)
    x = _make(gpu, 35, [3, 2], [20, 5], 16, 8, 16, torch.bfloat16, extra_rows=4)
    x["cu"] += 1
    if none == "blocks":
        x["kc"], x["vc"] = x["kc"][:0], x["vc"][:0]
    elif none == "columns":
        x["tables"] = x["tables"][:, :0].contiguous()
    else:
        x["ctx"].zero_()
    out = torch.full((9, 16, 128), 3.0, dtype=torch.bfloat16, device=gpu)
    assert _run(x, True, out=out) is out
    assert (out[1:6] == 0).all() and (out[0] == 3).all() and (out[6:] == 3).all()
