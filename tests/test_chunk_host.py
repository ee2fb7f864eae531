"""Chunks over the paged cache and rotary positions, on the host: the C entry points' refusals,
the page arithmetic, the frequencies' scaling rules (against transformers' where it is
installed)."""
import math

import pytest
import torch

from awesome_acceleration_amd import _lib, rotary


def _chunk(q=64, qs=2048, n=5, kc=64, vc=64, nb=4, bs=16, tab=64, mb=3, cu=64, ctx=64, cuk=None, B=2, mq=3, mk=0,
           hq=16, hkv=8, d=128, scale=0.1, causal=1, out=64, os=2048, ws=None, wb=0, dt=0):
    return _lib.lib().aac_prefill_paged(q, qs, n, kc, vc, nb, bs, tab, mb, cu, ctx, cuk, B, mq, mk, hq, hkv, d,
                                        scale, causal, out, os, ws, wb, dt, None)


def test_chunk_refusals():
    """Before any launch: every call here is refused on its arguments alone."""
    for a in (dict(dt=2), dict(dt=7), dict(d=64), dict(bs=7, mb=1 << 25)):
        assert _chunk(**a) == -2, a
    for a in (dict(n=-1), dict(B=-1), dict(hq=0), dict(mq=-1), dict(bs=0), dict(mb=0), dict(scale=0.0),
              dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(scale=2e38), dict(q=None), dict(out=None),
              dict(tab=None), dict(ctx=None), dict(kc=None), dict(vc=None), dict(nb=0), dict(nb=-1)):
        assert _chunk(**a) == -1, a
    for a in (dict(hq=12), dict(qs=2047 // 2), dict(os=1024), dict(cu=None, n=5), dict(n=1 << 31)):
        assert _chunk(**a) == -5, a
    for a in (dict(q=72), dict(kc=72), dict(vc=68), dict(out=2), dict(qs=2052), dict(os=2052)):
        assert _chunk(**a) == -3, a
    for a in (dict(n=0), dict(B=0), dict(mq=0)):
        assert _chunk(**a, q=None, kc=None) == 0, a


def test_rotary_refusals():
    def f(x=64, out=64, B=2, S=3, n=0, cu=None, h=4, d=128, cos=64, sin=64, rows=9, rot=64, td=2, dt=0):
        return _lib.lib().aac_rotary(x, 1, 1, 128, out, 1, 1, 128, B, S, n, cu, None, 0, h, d, cos, sin, rows, rot,
                                     0, 0, td, dt, None)

    for a in (dict(dt=3), dict(td=1), dict(td=9)):
        assert f(**a) == -2, a
    for a in (dict(rot=3), dict(rot=130), dict(d=127)):
        assert f(**a) == -5, a
    for a in (dict(d=0), dict(rot=-2), dict(rows=0), dict(rows=-1), dict(cos=None), dict(sin=None), dict(B=-1),
              dict(S=-1), dict(h=-1), dict(x=None), dict(out=None), dict(cu=64, n=-1)):
        assert f(**a) == -1, a
    for a in (dict(B=0), dict(S=0), dict(h=0), dict(cu=64, n=0)):
        assert f(**a, x=None) == 0, a

    def g(q=None, qo=None, k=64, v=64, kc=64, vc=64, tab=64, lens=64, B=2, sk=3, hkv=4, bs=16, mb=2, nb=5, rot=0):
        return _lib.lib().aac_rotary_append_paged(q, 1, 1, 128, k, 1, 1, 128, v, 1, 1, 128, qo, B, 3, sk, 0, None,
                                                  lens, None, 4, hkv, 128, None, None, 0, rot, 0, 0, kc, vc, nb, bs,
                                                  tab, mb, 0, 0, None)

    for a in (dict(k=None), dict(v=None), dict(kc=None), dict(vc=None), dict(tab=None), dict(lens=None), dict(q=64),
              dict(hkv=0), dict(bs=0), dict(mb=0), dict(nb=-1), dict(B=-1), dict(sk=-1), dict(rot=64)):
        assert g(**a) == -1, a
    assert g(B=0, k=None) == 0 and g(sk=0, k=None) == 0

    def t(f=64, n=8, start=0, rows=5, cos=64, sin=64, dt=0):
        return _lib.lib().aac_rotary_tables(f, n, None, start, rows, 1.0, cos, sin, dt, None)

    assert t(dt=3) == -2 and t(n=0) == -1 and t(rows=-1) == -1 and t(f=None) == -1 and t(cos=None) == -1
    assert t(cos=68) == -3 and t(start=(1 << 40) + 1) == -5 and t(rows=0, f=None) == 0
    assert t(rows=1 << 39) == -2


def test_page_of_a_key_by_multiplication():
    """x / d as x * ceil(2^(27 + s) / d) >> (27 + s) with s = ceil(log2 d), exact for x < 2^27."""
    import random
    r = random.Random(0)
    for d in [*range(1, 70), 255, 256, 257, (1 << 27) - 1, 1 << 27, *(r.randrange(1, 1 << 27) for _ in range(200))]:
        s = (d - 1).bit_length()
        m = -(-(1 << (27 + s)) // d)
        assert m < 1 << 32
        for k in [0, 1, 2, ((1 << 27) - 1) // d, *(r.randrange((1 << 27) // d + 1) for _ in range(20))]:
            for x in (k * d - 1, k * d, k * d + d - 1):
                if 0 <= x < 1 << 27:
                    assert x * m < 1 << 64 and (x * m) >> (27 + s) == x // d


def test_row_of_a_group_by_multiplication():
    """y / g as 2 y * ceil(2^31 / g) >> 32, exact for y, g < 2^15; a larger group is refused."""
    for g in [*range(1, 70), 255, 256, 257, 4095, 4096, (1 << 14) - 1, 1 << 14, (1 << 15) - 1]:
        m = -(-(1 << 31) // g)
        assert m < 1 << 32
        for y in {y for k in range((1 << 15) // g + 1) for y in (k * g - 1, k * g, k * g + g - 1)}:
            if 0 <= y < 1 << 15:
                assert (2 * y * m) >> 32 == y // g
    assert _chunk(hq=1 << 14, hkv=1, mq=1, qs=1 << 21, os=1 << 21) == -2


RULES = [
    dict(rope_type="linear", factor=4.0),
    dict(rope_type="dynamic", factor=4.0, original_max_position_embeddings=2048),
    dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768),
    dict(rope_type="yarn", factor=40.0, original_max_position_embeddings=4096, mscale=1.0, mscale_all_dim=0.8,
         beta_fast=16, beta_slow=2),
    dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=4096, attention_factor=1.5, truncate=False),
    dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
         original_max_position_embeddings=8192),
]


@pytest.mark.parametrize("rule", RULES, ids=lambda r: r["rope_type"])
@pytest.mark.parametrize("dim", [128, 64])
def test_scaled_frequencies_are_transformers(rule, dim):
    """transformers computes them in float32: 2^-18 apart at most (powers and logarithms of
    some tens of rounded steps, and its ramp's differences of near values)."""
    rope = pytest.importorskip("transformers.modeling_rope_utils")
    from transformers import LlamaConfig
    old = int(rule.get("original_max_position_embeddings", 4096))
    cfg = LlamaConfig(hidden_size=8 * dim, num_attention_heads=8, head_dim=dim, max_position_embeddings=old,
                      rope_parameters=dict(rule, rope_theta=1e6))
    fn = rope.ROPE_INIT_FUNCTIONS[rule["rope_type"]]
    n = 3 * old
    try:
        inv, factor = fn(cfg, torch.device("cpu"), seq_len=n)
    except (KeyError, AttributeError, TypeError) as e:
        pytest.skip(f"this transformers reads its configuration otherwise: {e!r}")
    got, f = rotary.scaled_frequencies(dim, 1e6, rule, n)
    assert got.dtype == torch.float64 and got.shape == (dim // 2,)
    assert abs(f - factor) < 1e-6
    assert ((got - inv.double()).abs() <= 2.0 ** -18 * got).all()


def test_scaling_refusals():
    f = rotary.scaled_frequencies
    base, one = f(8, 100.0)
    assert one == 1.0 and torch.allclose(base, 100.0 ** (-torch.arange(4, dtype=torch.float64) / 4))
    assert torch.equal(f(8, 100.0, {})[0], base) and torch.equal(f(8, 100.0, dict(rope_type="default"))[0], base)
    for match, a in (("unknown", dict(rope_type="longer", factor=2.0, original_max_position_embeddings=9)),
                     ("factor", dict(rope_type="linear")), ("1 or more", dict(rope_type="linear", factor=0.5)),
                     ("original_max", dict(rope_type="yarn", factor=2.0)),
                     ("low_freq", dict(rope_type="llama3", factor=2.0, original_max_position_embeddings=9)),
                     ("above", dict(rope_type="llama3", factor=2.0, original_max_position_embeddings=9,
                                    low_freq_factor=4, high_freq_factor=4))):
        with pytest.raises(RuntimeError, match=match):
            f(8, 100.0, a)
    for dim, theta in ((7, 9.0), (0, 9.0), (8, 0.0), (8, 1.0), (8, -2.0)):
        with pytest.raises(RuntimeError):
            f(dim, theta)
    with pytest.raises(RuntimeError, match="GPU"):
        rotary.RotaryEmbedding(8, device="cpu")
    with pytest.raises(RuntimeError, match="GPU"):
        rotary.apply_rotary_emb(torch.zeros(1, 1, 1, 8), torch.zeros(1, 4), torch.zeros(1, 4))


def test_engine_refuses_a_chunk_of_no_tokens_and_chunks_with_the_4_bit_cache():
    from awesome_acceleration_amd.llm import LLM
    for a in (dict(prefill_chunk=0), dict(prefill_chunk=-3), dict(prefill_chunk=2.5),
              dict(prefill_chunk=64, kv_cache_dtype="mxfp4")):
        with pytest.raises(ValueError, match="prefill_chunk"):
            LLM(**a)


DYNAMIC = dict(rope_type="dynamic", factor=4.0, original_max_position_embeddings=300)


@pytest.mark.parametrize("rule", [DYNAMIC, dict(type="dynamic", factor=4.0)], ids=["original", "model"])
def test_dynamic_scaling_leaves_the_original_context_as_it_is(rule):
    """transformers grows theta for a context past the original one alone; the model's tables
    are the unscaled ones, as far as the original context."""
    from awesome_acceleration_amd.qwen3 import Rope
    plain = Rope(64, 300, 1e4, "cpu", torch.float32)
    got = Rope(64, 300, 1e4, "cpu", torch.float32, rule)
    assert torch.equal(got.cos, plain.cos) and torch.equal(got.sin, plain.sin)
    longer = Rope(64, 4096, 1e4, "cpu", torch.float32, DYNAMIC)
    assert torch.equal(longer.cos, plain.cos) and torch.equal(longer.sin, plain.sin)
    with pytest.raises(RuntimeError, match="factor"):
        Rope(64, 300, 1e4, "cpu", torch.float32, dict(rope_type="dynamic"))
    transformers = pytest.importorskip("transformers.models.qwen3.modeling_qwen3")
    from transformers import Qwen3Config as Theirs
    try:
        theirs = transformers.Qwen3RotaryEmbedding(Theirs(
            hidden_size=64, num_attention_heads=1, head_dim=64, max_position_embeddings=300,
            rope_parameters=dict(DYNAMIC, rope_theta=1e4)))
        cos, sin = theirs(torch.zeros(1, 1, 64), torch.arange(300)[None])
    except (KeyError, AttributeError, TypeError) as e:
        pytest.skip(f"this transformers reads its configuration otherwise: {e!r}")
    # an angle of up to 299 in float32, its frequency's power rounded here and there: 4 units
    # of 2^-24 of it
    assert (got.cos - cos[0]).abs().max() <= 300 * 2.0 ** -22
    assert (got.sin - sin[0]).abs().max() <= 300 * 2.0 ** -22


def test_engine_refuses_dynamic_scaling_past_the_original_context():
    from awesome_acceleration_amd.llm import LLM
    from awesome_acceleration_amd.qwen3 import Qwen3Config
    for rule, limit in ((DYNAMIC, 300), (dict(type="dynamic", factor=2.0), 500)):
        cfg = Qwen3Config(num_hidden_layers=1, max_position_embeddings=500, rope_scaling=rule)
        with pytest.raises(ValueError, match=f"original {limit} tokens"):
            LLM(cfg, max_seq_len=limit + 1)


def test_config_files_name_their_scaling_either_way(tmp_path):
    """rope_scaling beside rope_theta, or rope_parameters with both in it, read as transformers
    reads them."""
    import json
    from awesome_acceleration_amd.qwen3 import Qwen3Config
    yarn = dict(rope_type="yarn", factor=2.0, original_max_position_embeddings=16384)
    linear = dict(type="linear", factor=4.0)

    def read(**data):
        path = tmp_path / "config.json"
        path.write_text(json.dumps(dict(hidden_size=512, max_position_embeddings=32768, **data)))
        c = Qwen3Config.from_json(path)
        assert c.hidden_size == 512 and c.max_position_embeddings == 32768
        return c.rope_theta, c.rope_scaling

    assert read() == (1e6, None)
    assert read(rope_theta=5e5) == (5e5, None)
    assert read(rope_theta=5e5, rope_scaling=None) == (5e5, None)
    assert read(rope_theta=5e5, rope_scaling=linear) == (5e5, linear)
    assert read(rope_scaling=dict(linear, rope_theta=3e5), rope_theta=5e5) == (3e5, linear)
    assert read(rope_parameters=dict(rope_type="default", rope_theta=2e4)) == (2e4, None)
    assert read(rope_parameters=dict(yarn, rope_theta=2e4)) == (2e4, yarn)
    assert read(rope_parameters=dict(yarn, rope_theta=2e4), rope_theta=5e5, rope_scaling=None) == (2e4, yarn)
    assert read(rope_parameters=yarn, rope_theta=5e5) == (5e5, yarn)
    assert read(rope_parameters=dict(yarn, rope_theta=2e4), rope_scaling=linear) == (1e6, linear)
    with pytest.raises(ValueError, match="layer type"):
        read(rope_parameters=dict(full_attention=yarn))
    with pytest.raises(ValueError, match="in part"):
        read(rope_parameters=dict(yarn, partial_rotary_factor=0.5))


def test_config_file_of_the_installed_transformers(tmp_path):
    transformers = pytest.importorskip("transformers")
    from awesome_acceleration_amd.qwen3 import Qwen3Config
    rule = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                original_max_position_embeddings=8192)
    try:
        theirs = transformers.Qwen3Config(rope_parameters=dict(rule, rope_theta=5e5))
    except (KeyError, AttributeError, TypeError) as e:
        pytest.skip(f"this transformers reads its configuration otherwise: {e!r}")
    theirs.save_pretrained(tmp_path)
    c = Qwen3Config.from_json(tmp_path / "config.json")
    assert c.rope_theta == 5e5 and c.rope_scaling == rule


def _engine(chunk=None, decode_fn=None):
    """The engine's loop alone: prompts of any length, every token a 7, no model or device."""
    import queue
    from types import SimpleNamespace
    from awesome_acceleration_amd import paged
    from awesome_acceleration_amd.llm import LLM
    llm = LLM.__new__(LLM)
    llm.config = SimpleNamespace(vocab_size=9, eos_token_id=0)
    llm.max_seq_len, llm.max_num_seqs, llm.block_size = 64, 3, 16
    llm.allocator = paged.BlockAllocator(12 + 1)
    llm.allocator.allocate(1)
    llm.use_graphs, llm.prefill_chunk, llm.decode_fn = False, chunk, decode_fn
    llm._request_queue, llm._loop_running, llm._loop_thread = queue.Queue(), False, None
    llm.stats = dict(decode_tokens=0)

    def chunk_step(filling):
        for s in filling:
            s.filled += chunk
        ended = [s for s in filling if s.filled >= len(s.req.token_ids[s.prompt_idx])]
        return torch.zeros(len(ended), 9), ended

    llm._prefill = llm._decode_step = lambda seqs: torch.zeros(len(seqs), 9)
    llm._prefill_chunk = chunk_step
    llm._sample_step = lambda seqs, logits, temperature: [7] * len(seqs)
    return llm


@pytest.mark.filterwarnings("ignore::pytest.PytestUnhandledThreadExceptionWarning")
@pytest.mark.parametrize("chunk", [None, 4])
@pytest.mark.parametrize("where", ["sample", "end of a prompt", "end"])
def test_a_step_that_fails_ends_every_request(chunk, where):
    """Whichever list its sequences are in, a caller gets the exception and does not wait on."""
    def fail(*a):
        raise MemoryError("no memory")

    llm = _engine(chunk, fail if where != "sample" else None)
    if where == "sample":
        llm._sample_step = fail
    n = 1 if where == "end of a prompt" else 3
    futs = [llm.generate([[2] * 3], max_tokens=n), llm.generate([[1] * 5, [3] * 30], max_tokens=9),
            llm.generate([[4] * 9] * 4, max_tokens=9)]
    for f in futs:
        with pytest.raises(MemoryError):
            f.result(timeout=20)
    llm._loop_thread.join(20)


@pytest.mark.parametrize("chunk", [None, 4])
def test_the_engines_loop_alone(chunk):
    llm = _engine(chunk, lambda tokens: "x" * len(tokens))
    futs = [llm.generate([[1] * 5, [2] * 3], max_tokens=2), llm.generate([[3] * 30] * 5, max_tokens=9)]
    got = [f.result(timeout=20) for f in futs]
    llm.stop()
    assert [[o.text for o in g] for g in got] == [["xx"] * 2, ["x" * 9] * 5]
    assert llm.allocator.num_free == 12


@pytest.mark.filterwarnings("ignore::pytest.PytestUnhandledThreadExceptionWarning")
@pytest.mark.parametrize("chunk", [None, 4])
def test_after_a_failed_step_the_engine_serves_again(chunk):
    """Blocks of the sequences that a failure ends go back to the pool."""
    llm = _engine(chunk)
    works = llm._decode_step

    def fail(seqs):
        raise MemoryError("no memory")

    for _ in range(3):
        llm._decode_step = fail
        with pytest.raises(MemoryError):
            llm.generate([[1] * 40] * 5, max_tokens=20).result(timeout=20)
        llm._loop_thread.join(20)
        assert llm.allocator.num_free == 12
        llm._decode_step = works
        assert [o.token_ids for o in llm.generate([[1] * 40] * 5, max_tokens=20).result(timeout=20)] == [[7] * 20] * 5
        assert llm.allocator.num_free == 12
    llm.stop()


@pytest.fixture
def launches(monkeypatch):
    """The names of a call's launches, none of which is made."""
    from awesome_acceleration_amd import flash_attn_interface as fai
    names = []
    for module in (fai, rotary):
        monkeypatch.setattr(module, "_on_gpu", lambda *ts: None)
    monkeypatch.setattr(fai, "_chunk_ws_bytes", lambda *a: 0)
    monkeypatch.setattr(_lib, "launch", lambda name, *a: names.append(name))
    return names


@pytest.mark.parametrize("turned", [False, True])
def test_what_the_attention_refuses_is_refused_before_the_append(launches, turned):
    from awesome_acceleration_amd import flash_attn_interface as fai

    def call(S=3, hq=4, hkv=2, d=128, bs=16, mb=2, nb=4, odd=0, **o):
        empty = torch.zeros(nb * bs * hkv * d + 8, dtype=torch.bfloat16)
        kc = empty[odd:odd + nb * bs * hkv * d].view(nb, bs, hkv, d)
        q = torch.zeros(1, dtype=torch.bfloat16).expand(2, S, hq, d)
        k = torch.zeros(2, S, hkv, d, dtype=torch.bfloat16)
        if turned:
            o["rotary_cos"] = o["rotary_sin"] = torch.zeros(9, d // 2)
        return fai.flash_attn_with_kvcache(q.contiguous(), kc, kc, k=k, v=k, cache_seqlens=1, causal=True,
                                           block_table=torch.zeros(2, mb, dtype=torch.int32), **o)

    call()
    assert launches == ["aac_rotary_append_paged", "aac_prefill_paged"]
    if turned:
        call(S=1)
        assert launches[2:] == ["aac_rotary_append_paged", "aac_decode_paged"]
    del launches[:]
    for S in (1, 3) if turned else (3,):
        for match, a in (("head_dim", dict(d=64)), ("head_dim", dict(d=256)), ("aligned", dict(odd=4))):
            with pytest.raises(RuntimeError, match=match):
                call(S, **a)
    for match, a in (("scale", dict(softmax_scale=2e38)), ("too many", dict(hq=1 << 14, hkv=1)),
                     ("names 2.27 tokens", dict(bs=7, mb=20_000_000))):
        with pytest.raises(RuntimeError, match=match):
            call(**a)
    assert launches == []
    call(mb=1, bs=7)
    assert len(launches) == 2


def test_rotary_refuses_2_32_threads():
    """Four waves a workgroup of 256 threads, 2^24 workgroups; the tables' threads a vector each."""
    def turn(n, h=1, d=128, dt=0, cu=64):
        return _lib.lib().aac_rotary(64, 0, h * d, d, 64, 0, h * d, d, 1, 0, n, cu, None, 0, h, d, 64, 64, 9, 2, 0,
                                     0, 2, dt, None)

    # a token a wave (rotary_dim 2: the element-wise kernel); n_seqs x seqlen as well
    for n in ((1 << 26) - 3, 1 << 26, 1 << 62):
        assert turn(n) == -2, n
    assert _lib.lib().aac_rotary(64, 0, 128, 128, 64, 0, 128, 128, 1 << 30, 1 << 30, 0, None, None, 0, 1, 128, 64, 64,
                                 9, 2, 0, 0, 2, 0, None) == -2

    def append(n, hq, rot=128):
        return _lib.lib().aac_rotary_append_paged(64, 0, hq * 128, 128, 64, 0, 512, 128, 64, 0, 512, 128, 64, 1, 0, 0,
                                                  n, 64, 64, None, hq, 4, 128, 64, 64, 9, rot, 0, 0, 64, 64, 1, 16, 64,
                                                  1, 2, 0, None)

    # 16-bit rows of 128 dims, sixteen a wave: 8 + 2 x 4 heads take one, 9 + 8 two, 65,528 + 8 4096
    for n, hq in (((1 << 26) - 3, 8), ((1 << 25) - 1, 9), (1 << 25, 9), (1 << 14, 65528)):
        assert append(n, hq) == -2, (n, hq)

    def tables(n, freqs, dt):
        return _lib.lib().aac_rotary_tables(64, freqs, None, 0, n, 1.0, 64, 64, dt, None)

    for n, freqs, dt in (((1 << 32) - 255, 4, 2), (1 << 32, 8, 0), ((1 << 28) - 15, 64, 2), (1 << 29, 64, 1)):
        assert tables(n, freqs, dt) == -2, (n, freqs)


@pytest.mark.filterwarnings("ignore::pytest.PytestUnhandledThreadExceptionWarning")
def test_a_failed_step_frees_no_block_of_another():
    """A block that a sequence gave back before the failure may be someone else's by then."""
    held, ended = [], []

    def text(tokens):
        ended.append(tokens)
        if len(ended) == 2:
            held.extend(llm.allocator.allocate(llm.allocator.num_free))
            raise MemoryError("no memory")
        return ""

    llm = _engine(decode_fn=text)
    with pytest.raises(MemoryError):
        llm.generate([[1] * 5, [2] * 5], max_tokens=2).result(timeout=20)
    llm._loop_thread.join(20)
    assert len(held) == 11 and llm.allocator.num_free == 1
