"""The 4-bit cache, the step maps and the log probabilities in the engine: the fused store
against the store of what it returns, every call of a run against the float64 oracle
(oracle/kv4.py), graph-captured decode against the eager loop, and the KV payload."""
import concurrent.futures

import numpy as np
import pytest
import torch

from awesome_acceleration_amd import fused, kv4, paged, qwen3
from awesome_acceleration_amd.llm import LLM, _Request, _Seq
from awesome_acceleration_amd.qwen3 import PagedKV4Cache, PagedKVCache, Qwen3Config
from oracle import kv4 as oracle4
from gpu_util import f64

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CFG = Qwen3Config(vocab_size=2048, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                  num_attention_heads=4, num_key_value_heads=2, head_dim=128,
                  max_position_embeddings=4096)


def _prompts(n, seed):
    rs = np.random.RandomState(seed)
    return [rs.randint(0, CFG.vocab_size, rs.randint(1, 150)).tolist() for _ in range(n)]


def _qkv_case(gpu, n, hq, hkv, dtype, seed):
    g = torch.Generator(device=gpu).manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device=gpu, dtype=torch.float32).to(DTYPES[dtype])  # noqa: E731
    wide = rnd(n, (hq + 2 * hkv) * 128 + 64)
    return dict(qkv=wide[:, :-64], q_norm_weight=rnd(128), k_norm_weight=rnd(128), eps=1e-6, cos=rnd(700, 128),
                sin=rnd(700, 128),
                positions=torch.randint(0, 700, (n,), generator=g, device=gpu, dtype=torch.int32))


# ---------------------------------------------------------------- fused store
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, hq, hkv", [(1, 1, 1), (5, 7, 1), (33, 6, 3), (600, 16, 8), (4099, 4, 2), (32801, 16, 8)])
def test_fused_store_is_the_store_of_what_it_returns(gpu, dtype, n, hq, hkv):
    print("case: fused store", dtype, n, hq, hkv, flush=True)
    a = _qkv_case(gpu, n, hq, hkv, dtype, n)
    nb = n // 48 + 2
    rs = np.random.RandomState(n)
    slots = rs.permutation(nb * 48)[:n]
    slots[3::7] = -1
    slots[4::9] = nb * 48
    slots = torch.from_numpy(slots).to(gpu)
    want = torch.randint(0, 256, (nb, hkv, 2, 48 * 68), dtype=torch.uint8, device=gpu)
    got, third = want.clone(), want.clone()
    args = dict(a)
    qkv = args.pop("qkv")
    q, k = kv4.qk_norm_rope_store_kv4(qkv, hq, **args, kv_cache=got, slot_mapping=slots)
    rq, rk = fused.qk_norm_rope_store(qkv, hq, hkv, **args)
    assert torch.equal(q, rq) and torch.equal(k, rk)
    kv4.kv4_store(k, qkv[:, (hq + hkv) * 128:].unflatten(1, (hkv, 128)), want, slots)
    assert torch.equal(got, want)  # every byte, also of the rows not named
    q2, none = kv4.qk_norm_rope_store_kv4(qkv, hq, **args, kv_cache=third, slot_mapping=slots, want_k=False)
    assert none is None and torch.equal(q2, q) and torch.equal(third, want)


@pytest.mark.parametrize("n", [1, 9, 5000])
def test_fused_append(gpu, n):
    print("case: fused append", n, flush=True)
    hq, hkv, bs, w = 8, 2, 16, 3
    a = _qkv_case(gpu, n, hq, hkv, "bf16", n)
    qkv = a.pop("qkv")
    rs = np.random.RandomState(n)
    nb = n * w
    tables = rs.permutation(nb).reshape(n, w).astype(np.int32)
    lens = rs.randint(0, w * bs, n).astype(np.int32)
    if n > 4:
        lens[1], lens[2] = w * bs, -1            # past the table: nothing is written
        tables[3], tables[4] = nb, -7            # outside the pool: nothing is written
    blk = tables[np.arange(n), np.clip(lens // bs, 0, w - 1)]
    ok = (lens >= 0) & (lens < w * bs) & (blk >= 0) & (blk < nb)
    slots = torch.from_numpy(np.where(ok, blk * bs + lens % bs, -1).astype(np.int64)).to(gpu)
    got, want = (torch.zeros((nb, hkv, 2, bs * 68), dtype=torch.uint8, device=gpu) for _ in "ab")
    kv4.qk_norm_rope_store_kv4(qkv, hq, **a, kv_cache=got, block_tables=torch.from_numpy(tables).to(gpu),
                               cache_seqlens=torch.from_numpy(lens).to(gpu))
    kv4.qk_norm_rope_store_kv4(qkv, hq, **a, kv_cache=want, slot_mapping=slots)
    assert torch.equal(got, want) and (got != 0).any()


def test_fused_store_refuses(gpu):
    a = _qkv_case(gpu, 5, 4, 2, "bf16", 0)
    cache = kv4.alloc_kv4_cache(2, 16, 2, device=gpu)
    slots = torch.arange(5, device=gpu)
    call = lambda **o: kv4.qk_norm_rope_store_kv4(**{**a, "n_q_heads": 4, "kv_cache": cache,  # noqa: E731
                                                     "slot_mapping": slots, **o})
    call()
    lens = torch.zeros(5, dtype=torch.int32, device=gpu)
    for bad in (dict(qkv=a["qkv"].float()), dict(n_q_heads=5), dict(q_norm_weight=a["q_norm_weight"][:64]),
                dict(k_norm_weight=a["k_norm_weight"].half()), dict(sin=a["sin"][:10]),
                dict(positions=a["positions"].long()), dict(slot_mapping=slots[:4]),
                dict(slot_mapping=slots.int()), dict(slot_mapping=None),
                dict(slot_mapping=None, block_tables=lens[:, None], cache_seqlens=lens[:3]),
                dict(slot_mapping=None, block_tables=lens[:3, None], cache_seqlens=lens),
                dict(kv_cache=cache.view(torch.int8)), dict(positions=a["positions"].cpu()),
                dict(qkv=a["qkv"][:, 1:], n_q_heads=4)):
        with pytest.raises(RuntimeError):
            call(**bad)


# ---------------------------------------------------------------- payload
def test_exported_rows_come_back_byte_for_byte(gpu):
    L, nb, hkv, bs, length = 3, 12, 2, 16, 75
    storage = kv4.alloc_kv4_cache(nb, bs, hkv, device=gpu, n_layers=L)
    g = torch.Generator(device=gpu).manual_seed(0)
    rows = torch.randn((2, L * nb * bs, hkv, 128), generator=g, device=gpu)
    rows *= torch.exp(8 * torch.randn((2, L * nb * bs, hkv, 1), generator=g, device=gpu))
    rows[:, 5::11] = 0
    rows[:, 6::11, :, 40] = torch.nan
    kv4.kv4_store(*rows, storage.flatten(0, 1), torch.arange(L * nb * bs, device=gpu))
    table = [7, 2, -1, 11, 0]
    for dt in (torch.bfloat16, torch.float32):
        k, v = kv4.kv4_export(storage, table, length, dtype=dt)
        assert k.shape == v.shape == (L, length, hkv, 128) and k.dtype == dt
        for i in range(L):
            at = [table[p // bs] * bs + p % bs if table[p // bs] >= 0 else -1 for p in range(length)]
            ref = oracle4.load(storage[i].cpu().numpy(), bs, at)
            assert np.array_equal(f64(k[i]), ref[0], equal_nan=True)
            assert np.array_equal(f64(v[i]), ref[1], equal_nan=True)
        back = storage.clone()
        kv4.kv4_import(k, v, back, table)  # onto themselves; the block outside the pool is skipped
        assert torch.equal(back, storage)
        other = torch.full_like(storage, 17)
        kv4.kv4_import(k, v, other, [3, 4, nb, 5, 6])
        # (what the bad block held is zeros here, and not written)
        k2, v2 = kv4.kv4_export(other, [3, 4, -1, 5, 6], length, dtype=dt)
        assert torch.equal(k2.nan_to_num(3), k.nan_to_num(3)) and torch.equal(v2.nan_to_num(3), v.nan_to_num(3))
        assert (other[:, [0, 1, 2, 7, 8, 9, 10, 11]] == 17).all()
    k, v = kv4.kv4_export(storage, [], 0)
    assert k.shape == (L, 0, hkv, 128)
    with pytest.raises(RuntimeError, match="too short"):
        kv4.kv4_export(storage, [1, 2], 33)


def test_payload_moves_between_the_caches(gpu):
    cfg = Qwen3Config(num_hidden_layers=3, num_key_value_heads=2, head_dim=128)
    wide = PagedKVCache(cfg, 8, 32, gpu, torch.bfloat16)
    g = torch.Generator(device=gpu).manual_seed(1)
    wide.storage.copy_(torch.randn(wide.storage.shape, generator=g, device=gpu))
    four, again = (PagedKV4Cache(cfg, 8, 32, gpu) for _ in "ab")
    payload = wide.export_request_kv([5, 1, 2], 70, seqlen=70)
    assert four.import_request_kv([0, 7, 3], payload, 70) == 70
    out = four.export_request_kv([0, 7, 3], 70, seqlen=71)
    assert len(out["layers"]) == 3 and out["layers"][0]["k"].dtype == torch.bfloat16
    for i, (a, b) in enumerate(zip(payload["layers"], out["layers"])):
        for n in "kv":
            want = oracle4.values(*oracle4.quantise(f64(a[n])))
            assert np.array_equal(f64(b[n]), want), (i, n)
    assert again.import_request_kv([0, 7, 3], out, 70) == 71
    assert torch.equal(again.storage, four.storage)
    assert wide.import_request_kv([5, 1, 2], out, 70) == 71
    for length in (71, -1):
        with pytest.raises(RuntimeError, match="tokens"):
            four.import_request_kv([0, 7, 3], out, length)
    with pytest.raises(ValueError, match="Layer count"):
        four.import_request_kv([0], {"layers": out["layers"][:1]}, 1)
    assert four.nbytes * 512 == wide.storage.numel() * 2 * 136


# ---------------------------------------------------------------- engine
def _run(prompts, max_tokens, logprobs=None, max_num_seqs=4, **o):
    llm = LLM(CFG, max_num_seqs=max_num_seqs, max_seq_len=256, block_size=32, seed=0, **o)
    each = logprobs if isinstance(logprobs, list) else [logprobs] * len(prompts)
    futs = [llm.generate([p], max_tokens=mt, ignore_eos=True, logprobs=k)
            for p, mt, k in zip(prompts, max_tokens, each)]
    outs = [f.result(timeout=120)[0] for f in futs]
    llm.stop()
    return llm, outs


MAX_TOKENS = [1, 5, 12, 3, 20, 8, 2, 15, 6]


@pytest.mark.parametrize("fused_layers", [True, False])
def test_engine_with_the_4_bit_cache(gpu, fused_layers, monkeypatch):
    """Every call that the engine makes, on the tensors it makes it with: stores are the
    oracle's bytes, attention is within the oracle's bound (as in the operator's own
    tests: bf16 probabilities twice 2^-8 of sum p |v|, the output's half step, 2^-16 for
    the float sums)."""
    print(f"case: engine, 4-bit cache, fused={fused_layers}", flush=True)
    seen = dict(store=0, attend=0)

    def check_attend(out, q, cache, tables, ctx):
        bs = cache.shape[3] // 68
        ref, absv, z = oracle4.decode(f64(q), cache.cpu().numpy(), bs, tables.cpu().numpy(), ctx.tolist(), 128 ** -0.5)
        lim = 2.0 ** -8 * np.abs(ref) + (2.0 ** -7 + 2.0 ** -16 * (1 + z)) * absv * (1 + 2.0 ** -8) + 2.0 ** -25
        assert (np.abs(f64(out).reshape(ref.shape) - ref) <= lim).all()
        seen["attend"] += 1

    def check_store(before, after, bs, k, v, slots):
        want = before.cpu().numpy()
        oracle4.store(want, bs, f64(k), f64(v), slots)
        assert np.array_equal(after.cpu().numpy(), want)
        seen["store"] += 1

    def rows_of(tables, lens, bs):
        return [int(t[p // bs]) * bs + p % bs for t, p in zip(tables.tolist(), lens.tolist())]

    real_fused, real_store = kv4.qk_norm_rope_store_kv4, kv4.kv4_store
    real_decode, real_append = kv4.decode_paged_kv4, kv4.flash_attn_with_kv4cache

    def fused_store(qkv, hq, *args, **o):
        cache = args[6]
        bs, hkv, before = cache.shape[3] // 68, cache.shape[1], cache.clone()
        q, k = real_fused(qkv, hq, *args, **o)
        rk = k if k is not None else fused.qk_norm_rope_store(qkv, hq, hkv, *args[:6])[1]
        slots = o["slot_mapping"].tolist() if "slot_mapping" in o else rows_of(o["block_tables"], o["cache_seqlens"], bs)
        check_store(before, cache, bs, rk, qkv[:, (hq + hkv) * 128:].unflatten(1, (hkv, 128)), slots)
        return q, k

    def store(k, v, cache, slots):
        before = cache.clone()
        real_store(k, v, cache, slots)
        check_store(before, cache, cache.shape[3] // 68, k, v, slots.tolist())

    def decode(q, cache, tables, ctx, **o):
        out = real_decode(q, cache, tables, ctx, **o)
        check_attend(out, q, cache, tables, ctx)
        return out

    def append(q, cache, **o):
        before = cache.clone()
        out = real_append(q, cache, **o)
        bs = cache.shape[3] // 68
        check_store(before, cache, bs, o["k"][:, 0], o["v"][:, 0], rows_of(o["block_table"], o["cache_seqlens"], bs))
        check_attend(out[:, 0], q[:, 0], cache, o["block_table"], o["cache_seqlens"] + 1)
        return out

    monkeypatch.setattr(kv4, "qk_norm_rope_store_kv4", fused_store)
    monkeypatch.setattr(kv4, "kv4_store", store)
    monkeypatch.setattr(kv4, "decode_paged_kv4", decode)
    monkeypatch.setattr(kv4, "flash_attn_with_kv4cache", append)
    prompts = _prompts(9, 0)
    o = dict(kv_cache_dtype="mxfp4", fused=fused_layers)
    llm, eager = _run(prompts, MAX_TOKENS, use_graphs=False, **o)
    assert isinstance(llm.cache, PagedKV4Cache)
    assert [x.generated_tokens for x in eager] == MAX_TOKENS and llm.allocator.num_free == 32
    steps = llm.stats["decode_steps"] * CFG.num_hidden_layers
    assert seen["attend"] == steps > 0
    assert seen["store"] == steps + llm.stats["prefill_calls"] * CFG.num_hidden_layers
    monkeypatch.undo()
    # a prompt attends to its own 16-bit K and V: its first token is the 16-bit cache's
    _, wide = _run(prompts, [1] * 9, use_graphs=False, fused=fused_layers)
    assert [x.token_ids[0] for x in wide] == [x.token_ids[0] for x in eager]
    # graph-captured decode (power-of-two buckets, padding rows, steps ahead) == eager
    _, graphed = _run(prompts, MAX_TOKENS, use_graphs=True, **o)
    assert [x.token_ids for x in graphed] == [x.token_ids for x in eager]


def test_engine_4_bit_batch_past_the_epilogue(gpu):
    """Enough sequences for the projection's epilogue form, which the 4-bit cache has not."""
    n = qwen3.QKV_ATTENTION_ROWS + 8
    prompts = _prompts(n, 4)
    o = dict(max_num_seqs=n, kv_cache_dtype="mxfp4")
    _, eager = _run(prompts, [6] * n, use_graphs=False, **o)
    _, graphed = _run(prompts, [6] * n, use_graphs=True, **o)
    assert [x.token_ids for x in graphed] == [x.token_ids for x in eager]


def _slack(x):
    return 2.0 ** -16 * (1 + np.abs(x))  # the operator's bound (test_gpu_logprobs.py)


@pytest.mark.parametrize("use_graphs", [False, True])
@pytest.mark.parametrize("kv", [None, "mxfp4"])
def test_engine_logprobs(gpu, use_graphs, kv, monkeypatch):
    """The scores are of the very logits that were sampled from, and reach the outputs of
    the requests that asked, token by token."""
    print(f"case: engine logprobs, graphs={use_graphs}, cache={kv}", flush=True)
    steps, real = [], LLM._scores

    def scores(self, logits, tok, top):
        out = real(self, logits, tok, top)
        if out is not None:
            steps.append((logits.clone(), tok.clone(), out))
        return out

    monkeypatch.setattr(LLM, "_scores", scores)
    prompts = _prompts(9, 2)
    asked = [0, 3, None, 32, 5, None, 1, 2, 7]
    llm, outs = _run(prompts, MAX_TOKENS, logprobs=asked, use_graphs=use_graphs, kv_cache_dtype=kv)
    assert steps
    known = set()
    for logits, tok, (lp, ent, top, ids) in steps:
        ref = oracle4.log_softmax(f64(logits))
        want = ref[np.arange(len(ref)), tok.cpu().numpy()]
        assert (np.abs(f64(lp) - want) <= _slack(want)).all()
        h = oracle4.entropy(f64(logits))
        assert (np.abs(f64(ent) - h) <= _slack(h)).all()
        assert np.array_equal(ids.numpy(), oracle4.top(f64(logits), ids.shape[1]))
        known.update(zip(tok.tolist(), lp.tolist(), ent.tolist()))
    for o, k, n in zip(outs, asked, MAX_TOKENS):
        if k is None:
            assert o.logprobs is None and o.entropies is None and o.top_logprobs is None
            continue
        assert len(o.logprobs) == len(o.entropies) == len(o.top_logprobs) == n
        assert [len(t) for t in o.top_logprobs] == [k] * n
        for t, lp, ent, top in zip(o.token_ids, o.logprobs, o.entropies, o.top_logprobs):
            assert (t, lp, ent) in known
            assert not top or top[0] == (t, lp)  # greedy: the token is the likeliest
    # the tokens do not depend on being asked
    _, plain = _run(prompts, MAX_TOKENS, use_graphs=use_graphs, kv_cache_dtype=kv)
    assert [x.token_ids for x in plain] == [x.token_ids for x in outs]


def test_engine_logprobs_of_sampled_tokens(gpu):
    llm = LLM(CFG, max_num_seqs=4, max_seq_len=256, block_size=32, seed=0)
    out = llm.generate(_prompts(3, 5), max_tokens=8, temperature=1.5, ignore_eos=True, logprobs=32).result(timeout=120)
    for o in out:
        for t, lp, top in zip(o.token_ids, o.logprobs, o.top_logprobs):
            assert lp <= top[0][1] and dict(top).get(t, lp) == lp
    for bad in (-1, 33, 2.0, "3"):
        with pytest.raises(ValueError, match="logprobs"):
            llm.generate([[1]], logprobs=bad)
    llm.stop()


def test_engine_prefill_maps_are_the_hosts(gpu):
    llm = LLM(CFG, max_num_seqs=4, max_seq_len=256, block_size=32, seed=0, use_graphs=False)
    lens = [1, 32, 33, 200]
    seqs = []
    rs = np.random.RandomState(0)
    free = (1 + rs.permutation(llm.cache.num_blocks - 1)).tolist()
    for i, n in enumerate(lens):
        req = _Request([[1] * n], 5, 0.0, True, concurrent.futures.Future())
        seqs.append(_Seq(req, 0, i, [free.pop() for _ in range(llm._blocks_for(n, 5))], [], n))
    got = llm._prefill_maps(lens, seqs)
    want = paged.build_prefill_metadata(lens, paged.pad_block_tables([s.blocks for s in seqs], 8), 32, gpu)
    assert all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(got, want))
    for block in (-1, llm.cache.num_blocks):
        seqs[2].blocks[1] = block
        with pytest.raises(IndexError):
            llm._prefill_maps(lens, seqs)


def test_the_operators_together(gpu):
    """A chunked prefill by hand: the maps take the blocks, the rows are stored through
    them, the last rows attend, and their logits are scored -- each on what the step
    before made."""
    rs = np.random.RandomState(7)
    bs, hq, hkv, vocab = 16, 8, 2, 999
    cached, new = [20, 0, 47, 3], [13, 40, 1, 0]
    n, T = 4, sum(new) + 5
    dev = lambda a, t=torch.int32: torch.tensor(a, dtype=t, device=gpu)  # noqa: E731
    tables = np.full((n, 4), -1, np.int32)
    for b, c in enumerate(cached):
        tables[b, :-(-c // bs)] = 20 + 4 * b + np.arange(-(-c // bs))
    gtables = torch.from_numpy(tables).to(gpu)
    maps = paged.build_step_maps(dev(new), dev(cached), gtables, bs, T, free_blocks=dev(list(range(19, 5, -1))))
    for b, c in enumerate(cached):  # the oracle's blocks: in order, sequence by sequence
        for j in range(-(-c // bs), -(-(c + new[b]) // bs)):
            tables[b, j] = 19 - (np.sum([-(-(x + y) // bs) - -(-x // bs) for x, y in
                                         zip(cached[:b], new[:b])], dtype=int) + j - -(-c // bs))
    assert np.array_equal(gtables.cpu().numpy(), tables)
    cache = np.zeros((36, hkv, 2, bs * 68), np.uint8)
    for b, c in enumerate(cached):
        p = np.arange(c)
        oracle4.store(cache, bs, rs.standard_normal((c, hkv, 128)), rs.standard_normal((c, hkv, 128)),
                      tables[b, p // bs] * bs + p % bs)
    gcache = torch.from_numpy(cache).to(gpu)
    k, v = (torch.from_numpy(rs.standard_normal((T, hkv, 128)).astype(np.float32)).bfloat16() for _ in "kv")
    slots = [int(tables[b, (c + i) // bs]) * bs + (c + i) % bs for b, c in enumerate(cached) for i in range(new[b])]
    assert maps.slot_mapping.tolist() == slots + [-1] * 5
    kv4.kv4_store(k.to(gpu), v.to(gpu), gcache, maps.slot_mapping)
    oracle4.store(cache, bs, f64(k), f64(v), slots)
    assert np.array_equal(gcache.cpu().numpy(), cache)
    q = torch.from_numpy(rs.standard_normal((n, hq, 128)).astype(np.float32)).bfloat16().to(gpu)
    out = kv4.decode_paged_kv4(q, gcache, gtables, maps.context_lens, max_context_len=64)
    ref, absv, z = oracle4.decode(f64(q), cache, bs, tables, [33, 40, 48, 3], 128 ** -0.5)
    lim = 2.0 ** -8 * np.abs(ref) + (2.0 ** -7 + 2.0 ** -16 * (1 + z)) * absv * (1 + 2.0 ** -8) + 2.0 ** -25
    assert (np.abs(f64(out) - ref) <= lim).all()
    head = torch.from_numpy(rs.standard_normal((hq * 128, vocab)).astype(np.float32)).to(gpu)
    logits = out.flatten(1).float() @ head
    tok = fused.argmax(logits)
    got = fused.token_logprobs(logits, tok, 5)
    want = oracle4.log_softmax(f64(logits))
    assert torch.equal(got.top_ids[:, 0], tok)
    assert np.array_equal(got.top_ids.cpu().numpy(), oracle4.top(f64(logits), 5))
    best = want[np.arange(n), tok.cpu().numpy()]
    assert (np.abs(f64(got.logprobs) - best) <= _slack(best)).all()
