"""The engine's chunked prefill and scaled rotary positions, and the chunk operators used
together, against the fp32 restatement of the model and plain computations."""
import numpy as np
import pytest
import torch

from awesome_acceleration_amd import flash_attn_interface as fai
from awesome_acceleration_amd import paged, rotary
from awesome_acceleration_amd.llm import LLM
from awesome_acceleration_amd.qwen3 import Qwen3Config
from oracle import qwen3_ref
from oracle.qwen3_ref import Qwen3Ref
from test_gpu_chunk import _check

pytestmark = pytest.mark.gpu

BASE = dict(vocab_size=2048, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
            num_attention_heads=4, num_key_value_heads=2, head_dim=128, max_position_embeddings=4096)
CFG = Qwen3Config(**BASE)


def _prompts(n, seed, most=300):
    rs = np.random.RandomState(seed)
    return [rs.randint(0, CFG.vocab_size, rs.randint(1, most)).tolist() for _ in range(n)]


def _run(prompts, max_tokens, cfg=CFG, **o):
    llm = LLM(cfg, **{**dict(max_num_seqs=4, max_seq_len=512, block_size=16, seed=0), **o})
    futs = [llm.generate([p], max_tokens=m, ignore_eos=True) for p, m in zip(prompts, max_tokens)]
    outs = [f.result(timeout=120)[0] for f in futs]
    llm.stop()
    return llm, outs


def _against_reference(llm, prompts, outs):
    ref = Qwen3Ref.from_model(llm.model)
    checked = total = 0
    for p, o in zip(prompts, outs):
        top2 = ref.logits(p + o.token_ids[:-1])[len(p) - 1:].topk(2, dim=-1)
        margin = top2.values[:, 0] - top2.values[:, 1]
        for i, tok in enumerate(o.token_ids):
            total += 1
            if margin[i] > 0.05:  # (bf16's noise, as in the engine's other tests)
                assert tok == int(top2.indices[i, 0]), f"token {i} of a prompt of {len(p)}"
                checked += 1
    assert checked >= 0.5 * total, checked


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("chunk", [1, 37, 128])
def test_prompts_in_chunks(gpu, fused, chunk, monkeypatch):
    """Tokens as the reference's, every attention call of the run as the float64 one's,
    and the graph engine's tokens the eager one's."""
    print("case: chunked engine", fused, chunk, flush=True)
    prompts = _prompts(7, chunk, 300 if chunk > 1 else 20)
    most = [1, 5, 12, 3, 20, 8, 2]
    calls, real = [], fai.prefill_paged

    def checked(q, kc, vc, cu, tables, ctx, max_q, **o):
        out = real(q, kc, vc, cu, tables, ctx, max_q, **o)
        new = cu.diff().tolist()
        assert o["max_context_len"] >= int(ctx.max()) and max_q == max(new)
        if len(calls) % 5 == 0:
            _check(out, dict(q=q, kc=kc, vc=vc, tables=tables, new=new, lens=ctx.tolist(), bs=kc.shape[1]), True)
        calls.append((new, ctx.tolist()))
        return out

    monkeypatch.setattr(fai, "prefill_paged", checked)
    llm, eager = _run(prompts, most, use_graphs=False, fused=fused, prefill_chunk=chunk)
    assert [o.generated_tokens for o in eager] == most
    assert calls and all(sum(new) <= chunk for new, _ in calls)
    assert llm.stats["prefill_tokens"] == sum(map(len, prompts))
    assert llm.allocator.num_free == llm.allocator.num_blocks - 1
    _against_reference(llm, prompts, eager)
    monkeypatch.setattr(fai, "prefill_paged", real)
    _, graphed = _run(prompts, most, use_graphs=True, fused=fused, prefill_chunk=chunk)
    assert [o.generated_tokens for o in graphed] == most
    _against_reference(llm, prompts, graphed)


def test_a_chunk_that_holds_every_prompt_changes_nothing(gpu):
    print("case: one chunk", flush=True)
    prompts = _prompts(4, 5)
    _, whole = _run(prompts, [6] * 4)
    _, chunked = _run(prompts, [6] * 4, prefill_chunk=4096)
    assert [o.token_ids for o in chunked] == [o.token_ids for o in whole]


def test_generation_goes_on_while_a_long_prompt_is_prefilled(gpu):
    """A short request admitted with a long one ends before the long prompt is in."""
    print("case: long prompt beside a short one", flush=True)
    llm = LLM(CFG, max_num_seqs=4, max_seq_len=4096, block_size=64, seed=0, prefill_chunk=32)
    short, long = [5, 6, 7], _prompts(1, 9, 3)[0] * 700
    outs = []
    futs = [llm.generate([p], max_tokens=m, ignore_eos=True, logprobs=2) for p, m in ((short, 8), (long, 3))]
    futs[0].add_done_callback(lambda f: outs.append(("short", futs[1].done())))
    got = [f.result(timeout=120)[0] for f in futs]
    llm.stop()
    assert outs == [("short", False)] and [o.generated_tokens for o in got] == [8, 3]
    assert len(got[1].logprobs) == 3 and len(got[0].top_logprobs[0]) == 2
    _against_reference(llm, [short, long], got)


@pytest.mark.parametrize("rule", [dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=64),
                                  dict(rope_type="linear", factor=3.0), None], ids=["yarn", "linear", "none"])
def test_model_with_scaled_positions(gpu, rule, monkeypatch):
    print("case: rope scaling", rule, flush=True)
    cfg = Qwen3Config(**{**BASE, "max_position_embeddings": 256}, rope_scaling=rule)

    def tables(positions, head_dim, theta):
        f, size = rotary.scaled_frequencies(head_dim, theta, rule)
        a = positions.double()[:, None].cpu() * f
        a = torch.cat((a, a), -1)
        return tuple((size * t).float().to(positions.device) for t in (a.cos(), a.sin()))

    monkeypatch.setattr(qwen3_ref, "rope_tables", tables)
    prompts = _prompts(4, 3, 200)
    llm, outs = _run(prompts, [8] * 4, cfg=cfg, prefill_chunk=50)
    _against_reference(llm, prompts, outs)
    # the tables reach as far as the scaled context
    assert llm.model.rope.cos.shape[0] == (256 if rule is None or rule["rope_type"] == "yarn" else 768)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_operators_together(gpu, dtype):
    """A server's two steps over one cache: packed prompts rotated, stored and attended in
    chunks, then draft tokens through the kvcache call; captured and replayed like eager."""
    print("case: together", dtype, flush=True)
    hq, hkv, bs = 8, 2, 16
    lens, g = [70, 3, 129], torch.Generator(device=gpu).manual_seed(1)
    rope = rotary.RotaryEmbedding(64, 1e6, dict(rope_type="yarn", factor=2.0, original_max_position_embeddings=64),
                                  device=gpu)
    cos, sin = rope.cos_sin(256, dtype=dtype)
    tables = torch.randperm(30, generator=g, device=gpu)[:30].view(3, 10).to(torch.int32)
    kc, vc = paged.alloc_kv_cache(30, bs, hkv, 128, dtype=dtype, device=gpu)
    rnd = lambda n: torch.randn((n, hq + 2 * hkv, 128), generator=g, device=gpu).to(dtype)  # noqa: E731
    done, x = [0, 0, 0], {}
    for step in ([50, 0, 64], [20, 3, 65]):
        held = torch.tensor(done, dtype=torch.int32, device=gpu)
        new = torch.tensor(step, dtype=torch.int32, device=gpu)
        maps = paged.build_step_maps(new, held, tables, bs, sum(step))
        q, k, v = rnd(sum(step)).split((hq, hkv, hkv), 1)
        qr = rotary.rotary_append_paged(q, k, v, kc, vc, tables, held, cos, sin, cu_seqlens=maps.cu_seqlens)
        assert torch.equal(vc.view(-1, hkv, 128)[maps.slot_mapping], v)
        at = cos[maps.positions], sin[maps.positions]
        assert torch.equal(kc.view(-1, hkv, 128)[maps.slot_mapping],
                           rotary.apply_rotary_emb(k[:, None], *at, seqlen_offsets=torch.arange(
                               sum(step), dtype=torch.int32, device=gpu))[:, 0])
        out = fai.prefill_paged(qr, kc, vc, maps.cu_seqlens, tables, maps.context_lens, max(step))
        done = [a + b for a, b in zip(done, step)]
        x = dict(q=qr, kc=kc, vc=vc, tables=tables, new=step, lens=done, bs=bs)
        _check(out, x, True, what=f"step {step}")
    assert done == lens
    # three draft tokens each, captured
    rows = rnd(9).view(3, 3, hq + 2 * hkv, 128)
    held = torch.tensor(done, dtype=torch.int32, device=gpu)

    def draft():
        q, k, v = rows.split((hq, hkv, hkv), 2)
        return fai.flash_attn_with_kvcache(q, kc, vc, k=k, v=v, rotary_cos=cos, rotary_sin=sin, cache_seqlens=held,
                                           block_table=tables, causal=True, rotary_interleaved=False)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        draft()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = draft()
    for n in range(3):
        rows.copy_(rnd(9).view(rows.shape))
        held.copy_(torch.tensor(done, device=gpu))
        graph.replay()
        got, cache = out.clone(), kc.clone()
        assert torch.equal(draft(), got) and torch.equal(kc, cache)
        q = rotary.apply_rotary_emb(rows[:, :, :hq], cos, sin, seqlen_offsets=held)
        _check(got.view(-1, hq, 128), dict(q=q.reshape(-1, hq, 128), kc=kc, vc=vc, tables=tables, new=[3] * 3,
                                           lens=[d + 3 for d in done], bs=bs), True, what=f"draft {n}")
        done = [d + n for d in done]  # some of them are kept


@pytest.mark.parametrize("rule", [dict(rope_type="dynamic", factor=4.0, original_max_position_embeddings=512),
                                  dict(type="dynamic", factor=2.0),
                                  dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                                       original_max_position_embeddings=64)],
                         ids=["dynamic", "dynamic-model", "llama3"])
def test_model_with_more_scaled_positions(gpu, rule, monkeypatch):
    """(Contexts within the original one: dynamic scaling leaves them as they are.)"""
    print("case: rope scaling", rule, flush=True)
    cfg = Qwen3Config(**{**BASE, "max_position_embeddings": 512}, rope_scaling=rule)

    def tables(positions, head_dim, theta):
        f = theta ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
        if rule.get("rope_type") == "llama3":
            f, _ = rotary.scaled_frequencies(head_dim, theta, rule)
        a = positions.double()[:, None].cpu() * f
        a = torch.cat((a, a), -1)
        return tuple(t.float().to(positions.device) for t in (a.cos(), a.sin()))

    monkeypatch.setattr(qwen3_ref, "rope_tables", tables)
    prompts = _prompts(4, 3, 200)
    llm, outs = _run(prompts, [8] * 4, cfg=cfg, prefill_chunk=50)
    _against_reference(llm, prompts, outs)
