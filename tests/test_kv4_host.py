"""The 4-bit cache, the step maps and the token log probabilities without a GPU: the
oracle's format against a search over the grid, and the refusals of every entry
point, which come before any launch."""
import numpy as np
import pytest
import torch

from awesome_acceleration_amd import _lib, fused, kv4, paged
from oracle import kv4 as oracle4

P = 1 << 20  # a placeholder address, never read


def test_quantise_takes_the_nearest_value_and_the_stated_scale():
    rs = np.random.RandomState(0)
    x = rs.standard_normal((50, 128)) * np.exp(rs.uniform(-60, 60, (50, 1)))
    x[0] = 0.0
    codes, scales = oracle4.quantise(x)
    got = oracle4.values(codes, scales)
    for r in range(50):
        for b in range(4):
            blk = x[r, 32 * b:32 * b + 32]
            a = np.abs(blk).max()
            e = int(scales[r, b]) - 127
            if a:
                n = int(np.floor(np.log2(a)))
                assert e == n - 2 + (a >= 1.75 * 2.0 ** n)
            grid = np.concatenate((oracle4.GRID, -oracle4.GRID)) * 2.0 ** e
            d = np.abs(blk[:, None] - grid).min(-1)
            assert np.array_equal(np.abs(got[r, 32 * b:32 * b + 32] - blk), d)


def test_quantise_ties_bounds_and_bad_blocks():
    x = np.zeros((6, 128))
    x[0, :9] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, -0.25, -2.5]  # scale 1: ties to the even code
    x[1, 0], x[1, 40] = 6.99, 7.0                                   # stays at 6, becomes 4 x 2
    x[2, 0] = 2.0 ** 127.9                                          # past the largest scale
    x[3, 0] = 2.0 ** -140                                           # below the smallest
    x[4, 0], x[5, 127] = np.inf, np.nan
    codes, scales = oracle4.quantise(x)
    v = oracle4.values(codes, scales)
    assert v[0, :9].tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 0.0, -2.0]
    assert v[1, 0] == 6.0 and v[1, 40] == 8.0
    assert scales[2, 0] == 252 and v[2, 0] == 6.0 * 2.0 ** 125
    assert scales[3, 0] == 2 and v[3, 0] == 0.0
    assert scales[4].tolist()[0] == 255 and np.isnan(v[4, :32]).all() and (v[4, 32:] == 0).all()
    assert scales[5, 3] == 255 and np.isnan(v[5, 96:]).all()


def test_pack_and_rows_round_trip():
    rs = np.random.RandomState(1)
    cache = np.zeros((3, 2, 2, 16 * 68), np.uint8)
    k, v = rs.standard_normal((5, 2, 128)), rs.standard_normal((5, 2, 128))
    slots = [7, -1, 47, 48, 0]
    oracle4.store(cache, 16, k, v, slots)
    kl, vl = oracle4.load(cache, 16, slots)
    want = oracle4.values(*oracle4.quantise(k))
    for t in (0, 2, 4):
        assert np.array_equal(kl[t], want[t])
    assert (kl[[1, 3]] == 0).all() and (vl[[1, 3]] == 0).all()


def _store(**o):
    a = dict(k=P, v=P, ks=1024, vs=1024, c=P, nb=4, bs=16, s=P, n=4, h=8, d=128, dt=0)
    a.update(o)
    return _lib.lib().aac_kv4_store(*a.values(), None)


@pytest.mark.parametrize("change, code", [
    (dict(k=None), -1), (dict(v=None), -1), (dict(c=None), -1), (dict(s=None), -1), (dict(n=-1), -1),
    (dict(nb=0), -1), (dict(bs=0), -1), (dict(h=0), -1), (dict(dt=9), -2), (dict(d=64), -2),
    (dict(bs=24), -5), (dict(ks=1000), -5), (dict(vs=1000), -5), (dict(c=P + 16), -3),
    (dict(k=P + 1), -3), (dict(n=0, k=None), 0)])
def test_store_refusals(change, code):
    assert _store(**change) == code


@pytest.mark.parametrize("change, code", [
    (dict(k=None), -1), (dict(t=None), -1), (dict(l=None), -1), (dict(w=0), -1), (dict(n=-1), -1),
    (dict(bs=8), -5), (dict(ks=1000), -5), (dict(dt=3), -2), (dict(c=P + 32), -3), (dict(n=0), 0)])
def test_append_refusals(change, code):
    a = dict(k=P, v=P, ks=1024, vs=1024, c=P, nb=4, bs=16, t=P, w=3, l=P, n=4, h=8, d=128, dt=0)
    a.update(change)
    assert _lib.lib().aac_kv4_append(*a.values(), None) == code


@pytest.mark.parametrize("change, code", [
    (dict(c=None), -1), (dict(s=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(n=-1), -1),
    (dict(k=P + 8), -3), (dict(bs=20), -5), (dict(d=64), -2), (dict(dt=-1), -2), (dict(n=0), 0)])
def test_load_refusals(change, code):
    a = dict(c=P, nb=4, bs=16, s=P, n=4, h=8, d=128, k=P, v=P, dt=0)
    a.update(change)
    assert _lib.lib().aac_kv4_load(*a.values(), None) == code


@pytest.mark.parametrize("change, code", [
    (dict(q=None), -1), (dict(c=None), -1), (dict(t=None), -1), (dict(l=None), -1), (dict(o=None), -1),
    (dict(n=-1), -1), (dict(w=0), -1), (dict(hq=0), -1), (dict(hq=12), -5), (dict(hq=136, qs=17408, os=17408), -2),
    (dict(d=64), -2), (dict(dt=3), -2), (dict(n=70000), -2), (dict(qs=1000), -5), (dict(os=1000), -5),
    (dict(q=P + 8), -3), (dict(qs=2052), -3), (dict(o=P + 4), -3), (dict(bs=17), -5), (dict(c=P + 8), -3),
    (dict(part=128, w=64), -4), (dict(part=128, w=64, ws=P, wsb=1 << 10), -4),
    (dict(part=128, w=64, ws=P + 8, wsb=1 << 30), -3), (dict(n=0), 0), (dict(k=P), -1), (dict(v=P), -1),
    (dict(k=P, v=P, ks=1000, vs=1024), -5), (dict(k=P + 1, v=P, ks=1024, vs=1024), -3)])
def test_decode_refusals(change, code):
    a = dict(q=P, qs=2048, k=None, v=None, ks=0, vs=0, c=P, nb=4, bs=16, t=P, w=3, l=P, n=4, mcl=0, hq=16, h=8, d=128,
             scale=1.0, o=P, os=2048, ws=None, wsb=0, part=0, dt=0)
    a.update(change)
    assert _lib.lib().aac_kv4_decode(*a.values(), None) == code


def test_decode_workspace_is_what_the_plan_writes():
    f = _lib.lib().aac_kv4_decode_workspace_bytes
    assert f(4, 16, 8, 128, 16, 3, 0, 0) == 0
    # 64 blocks of 16 in 256-token partitions: 4 partitions x (128 + 1) floats
    assert f(3, 16, 8, 128, 16, 64, 0, 256) == 3 * 16 * 4 * 129 * 4
    assert f(3, 16, 8, 128, 16, 64, 256, 256) == 0
    assert f(0, 16, 8, 128, 16, 64, 0, 256) == 0


@pytest.mark.parametrize("change, code", [
    (dict(new=None), -1), (dict(t=None), -1), (dict(ctx=None), -1), (dict(cu=None), -1),
    (dict(taken=None), -1), (dict(pos=None), -1), (dict(slots=None), -1), (dict(n=-1), -1),
    (dict(w=0), -1), (dict(bs=0), -1), (dict(f=None), -1), (dict(nf=-1), -1), (dict(tok=-1), -1),
    (dict(n=8193), -2), (dict(tok=1 << 31), -2)])
def test_step_maps_refusals(change, code):
    a = dict(new=P, cached=None, t=P, n=4, w=3, bs=16, f=P, nf=5, tok=10, cu=P, pos=P, slots=P, ctx=P,
             taken=P)
    a.update(change)
    assert _lib.lib().aac_step_maps(*a.values(), None) == code


@pytest.mark.parametrize("change, code", [
    (dict(x=None), -1), (dict(t=None), -1), (dict(lp=None), -1), (dict(h=None), -1), (dict(tl=None), -1),
    (dict(ti=None), -1), (dict(rows=-1), -1), (dict(cols=0), -1), (dict(stride=99), -1), (dict(k=-1), -1),
    (dict(k=33), -2), (dict(cols=(1 << 20) + 1, stride=1 << 21), -2), (dict(dt=3), -2),
    (dict(cols=3, k=4), -5), (dict(x=P + 1), -3), (dict(ws=None), -4), (dict(wsb=8), -4),
    (dict(ws=P + 8), -3), (dict(rows=0), 0)])
def test_token_logprobs_refusals(change, code):
    a = dict(x=P, stride=100, rows=4, cols=100, t=P, k=5, lp=P, h=P, tl=P, ti=P, ws=P, wsb=1 << 20, dt=0)
    a.update(change)
    assert _lib.lib().aac_token_logprobs(*a.values(), None) == code


def test_alloc_refuses_shapes_the_kernels_are_not_built_for():
    c = kv4.alloc_kv4_cache(3, 32, 2, device="cpu", n_layers=2)
    assert c.shape == (2, 3, 2, 2, 32 * 68) and c.dtype == torch.uint8 and not c.any()
    with pytest.raises(RuntimeError, match="multiple of 16"):
        kv4.alloc_kv4_cache(3, 24, 2, device="cpu")
    with pytest.raises(RuntimeError, match="head_dim"):
        kv4.alloc_kv4_cache(3, 32, 2, 64, device="cpu")


def test_every_surface_refuses_host_tensors():
    c = kv4.alloc_kv4_cache(3, 32, 2, device="cpu")
    k = torch.zeros(4, 2, 128)
    i64, i32 = torch.zeros(4, dtype=torch.int64), torch.zeros(4, dtype=torch.int32)
    t = torch.zeros(4, 2, dtype=torch.int32)
    for f in (lambda: kv4.kv4_store(k, k, c, i64), lambda: kv4.kv4_load(c, i64),
              lambda: kv4.decode_paged_kv4(k, c, t, i32),
              lambda: kv4.flash_attn_with_kv4cache(k[:, None], c, cache_seqlens=i32, block_table=t),
              lambda: paged.build_step_maps(i32, i32, t, 16, 4),
              lambda: fused.token_logprobs(torch.zeros(4, 9), i64)):
        with pytest.raises(RuntimeError, match="GPU"):
            f()


def test_top_orders_ties_nan_and_signed_zeros():
    x = np.array([[1.0, np.nan, 1.0, -0.0, 0.0, -np.inf]])
    assert oracle4.top(x, 6).tolist() == [[1, 0, 2, 3, 4, 5]]


@pytest.mark.parametrize("change, code", [
    (dict(x=None), -1), (dict(qw=None), -1), (dict(kw=None), -1), (dict(cos=None), -1), (dict(sin=None), -1),
    (dict(pos=None), -1), (dict(q=None), -1), (dict(c=None), -1), (dict(s=None), -1), (dict(n=-1), -1),
    (dict(hq=0), -1), (dict(h=0), -1), (dict(maxp=0), -1), (dict(nb=0), -1), (dict(d=64), -2), (dict(dt=2), -2),
    (dict(dt=7), -2), (dict(bs=24), -5), (dict(xs=4095), -5), (dict(xs=4100), -3), (dict(c=P + 16), -3),
    (dict(x=P + 8), -3), (dict(k=P + 8), -3), (dict(qw=P + 2), -3), (dict(s=None, t=P, l=P, w=0), -1),
    (dict(s=None, t=P, w=2), -1), (dict(s=None, l=P, w=2), -1), (dict(n=0, x=None), 0)])
def test_fused_store_refusals(change, code):
    a = dict(x=P, xs=4096, n=4, hq=16, h=8, d=128, qw=P, kw=P, eps=1e-6, cos=P, sin=P, maxp=100, pos=P, q=P,
             k=None, c=P, nb=4, bs=16, s=P, t=None, w=0, l=None, dt=0)
    a.update(change)
    assert _lib.lib().aac_qk_norm_rope_store_kv4(*a.values(), None) == code


def test_engine_refuses_an_unknown_cache_type():
    from awesome_acceleration_amd.llm import LLM
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        LLM(kv_cache_dtype="int8")


def test_sizes_past_32_bit_offsets_are_refused():
    big = 1 << 23
    assert _store(bs=2 * big) == _store(bs=big + 16) == -2 and _store(bs=big, n=0) == 0
    # 2^24 workgroups of 256 threads: 16 tokens of two heads each
    assert _store(n=16 << 24, h=1) == _store(n=4 << 24, h=8) == -2
    L = _lib.lib()
    assert L.aac_kv4_load(P, 4, 16, P, 4 << 24, 8, 128, P, P, 0, None) == -2
    a = (P, 1 << 26, 16, 8, 128, P, P, 1e-6, P, P, 100, P, P, None, P, 4, 16, P, None, 0, None, 0, None)
    assert L.aac_qk_norm_rope_store_kv4(P, 4096, *a[1:]) == -2
    assert L.aac_token_logprobs(P, 100, 1 << 24, 100, P, 0, P, P, P, P, P, 1 << 40, 0, None) == -2
    # a table's capacity passes 2^31 tokens: the plan stays within it (64 partitions of 2^25)
    assert L.aac_kv4_decode_workspace_bytes(1, 1, 1, 128, big, 1 << 20, 0, 0) == 64 * 129 * 4


def test_oracle_decode_is_torchs_attention_over_the_values():
    rs = np.random.RandomState(2)
    bs, hkv, hq, lens = 16, 2, 6, [5, 33, 0]
    tables = rs.permutation(9).reshape(3, 3)
    cache = np.full((9, hkv, 2, bs * 68), 255, np.uint8)
    kv = {}
    for b, n in enumerate(lens):
        p = np.arange(n)
        kv[b] = rs.standard_normal((2, n, hkv, 128))
        oracle4.store(cache, bs, *kv[b], tables[b, p // bs] * bs + p % bs)
    q = rs.standard_normal((3, hq, 128))
    out, absv, _ = oracle4.decode(q, cache, bs, tables, lens, 0.09)
    for b, n in enumerate(lens):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        k, v = (torch.from_numpy(oracle4.values(*oracle4.quantise(x))).transpose(0, 1).repeat_interleave(3, 0)
                for x in kv[b])
        att = lambda v: torch.nn.functional.scaled_dot_product_attention(  # noqa: E731
            torch.from_numpy(q[b])[:, None], k, v, scale=0.09)[:, 0].numpy()
        assert np.allclose(out[b], att(v), rtol=1e-12, atol=1e-13)
        assert np.allclose(absv[b], att(v.abs()), rtol=1e-12, atol=1e-13)


def test_oracle_scores_are_torchs():
    rs = np.random.RandomState(3)
    x = rs.standard_normal((6, 200)) * 5
    x[1, :150] = -np.inf
    x[2] = np.round(x[2])  # equal values
    t = torch.from_numpy(x)
    assert np.allclose(oracle4.log_softmax(x), torch.log_softmax(t, -1).numpy(), rtol=1e-13)
    assert np.allclose(oracle4.entropy(x), torch.distributions.Categorical(logits=t).entropy().numpy(), rtol=1e-12)
    # the first index first among equals: a stable sort
    order = torch.sort(t, dim=-1, descending=True, stable=True).indices.numpy()
    assert np.array_equal(oracle4.top(x, 20), order[:, :20])
    x[4, 7] = np.nan
    assert oracle4.top(x, 1)[4, 0] == 7 == int(torch.from_numpy(x[4]).argmax())


def test_limits_are_the_headers():
    import re
    from pathlib import Path
    text = (Path(__file__).parent.parent / "include" / "aac_attn.h").read_text()
    limit = lambda name: eval(re.search(rf"#define {name} (.+)", text)[1])  # noqa: E731
    assert limit("AAC_STEP_MAPS_MAX_SEQS") == paged.MAX_MAP_SEQS
    assert limit("AAC_LOGPROBS_MAX_TOP") == fused.MAX_TOP_LOGPROBS
    assert limit("AAC_LOGPROBS_MAX_COLS") == fused.MAX_LOGPROB_COLS


@pytest.mark.parametrize("call", ["decode", "append", "logprobs"])
def test_workspaces_live_until_the_library_has_returned(call, monkeypatch):
    """Other threads get the interpreter and the allocator while the library enqueues its
    launches: every buffer that a call allocates for it is held until then."""
    import weakref
    made, entered = [], []
    empty = torch.empty

    def recorded(*a, **o):
        t = empty(*a, **o)
        made.append((t.data_ptr(), weakref.ref(t)))
        return t

    def launch(name, device, *args):
        held = {at: ref() is not None for at, ref in made if at}
        entered.append([held[a] for a in args if a in held])

    monkeypatch.setattr(torch, "empty", recorded)
    monkeypatch.setattr(_lib, "launch", launch)
    for module in (kv4, fused):
        monkeypatch.setattr(module, "_on_gpu", lambda *ts: None)
    cache = kv4.alloc_kv4_cache(70, 32, 2, device="cpu")
    q, t = torch.zeros(4, 2, 128), torch.zeros(4, 64, dtype=torch.int32)
    lens = torch.full((4,), 2000, dtype=torch.int32)
    if call == "decode":
        kv4.decode_paged_kv4(q, cache, t, lens, partition_tokens=256)
    elif call == "append":
        kv4.flash_attn_with_kv4cache(q[:, None], cache, k=q[:, None], v=q[:, None], cache_seqlens=lens,
                                     block_table=t)
    else:
        fused.token_logprobs(torch.zeros(4, 100), torch.zeros(4, dtype=torch.int64), 3)
    (held,) = entered
    # the workspace and the outputs of torch.empty (one; log probabilities two)
    assert held == [True] * (3 if call == "logprobs" else 2)


def test_fused_store_refuses_2_32_threads():
    """A wave a token, four a workgroup: 2^24 workgroups of 256 threads from 2^26 - 3 tokens on."""
    L = _lib.lib()
    call = lambda n, nb: L.aac_qk_norm_rope_store_kv4(  # noqa: E731
        P, 4096, n, 16, 8, 128, P, P, 1e-6, P, P, 100, P, P, None, P, nb, 16, P, None, 0, None, 0, None)
    for n in ((1 << 26) - 3, (1 << 26) - 1, 1 << 26):
        assert call(n, 0) == -2, n
    assert call((1 << 26) - 4, 0) == -1  # (of the cache: one token fewer is not refused for its number)


@pytest.mark.parametrize("splits, most, part", [(0, None, 0), (1, None, 64 * 32), (3, None, 683), (4, 1000, 250),
                                                (5000, None, 1), (2, 1 << 40, 1024)])
def test_num_splits_and_lengths_as_the_16_bit_call_takes_them(splits, most, part, monkeypatch):
    calls = []
    monkeypatch.setattr(_lib, "launch", lambda name, device, *args: calls.append(args))
    monkeypatch.setattr(kv4, "_on_gpu", lambda *ts: None)
    cache, q = kv4.alloc_kv4_cache(70, 32, 2, device="cpu"), torch.zeros(4, 1, 2, 128)
    table = torch.zeros(64, 4, dtype=torch.int32).t()
    a = dict(block_table=table, num_splits=splits, max_context_len=most, causal=True)
    kv4.flash_attn_with_kv4cache(q, cache, cache_seqlens=9, **a)
    kv4.flash_attn_with_kv4cache(q, cache, cache_seqlens=torch.full((4,), 9, dtype=torch.int32), **a)
    assert calls[0][-2] == calls[1][-2] == part
    with pytest.raises(RuntimeError, match="cache_seqlens"):
        kv4.flash_attn_with_kv4cache(q, cache, cache_seqlens=torch.full((4,), 9), **a)


def test_a_cache_of_no_heads_is_refused(monkeypatch):
    monkeypatch.setattr(kv4, "_on_gpu", lambda *ts: None)
    cache, q = torch.zeros(3, 0, 2, 32 * 68, dtype=torch.uint8), torch.zeros(4, 2, 128)
    t, lens = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="KV heads"):
        kv4.decode_paged_kv4(q, cache, t, lens)
    with pytest.raises(RuntimeError, match="KV heads"):
        kv4.flash_attn_with_kv4cache(q[:, None], cache, cache_seqlens=lens, block_table=t)
