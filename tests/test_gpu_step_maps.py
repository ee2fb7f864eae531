"""Step maps built on the GPU against the host's metadata construction and allocator."""
import numpy as np
import pytest
import torch

from awesome_acceleration_amd import paged

pytestmark = pytest.mark.gpu


def _i32(x, gpu):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


def _host(new, cached, tables, bs, n_tokens, free):
    """The same in plain Python."""
    tables = tables.copy()
    n, w = tables.shape
    new, cached = [max(0, x) for x in new], [max(0, x) for x in cached]
    taken = 0
    if free is not None:
        for b in range(n):
            held, want = min(w, -(-cached[b] // bs)), min(w, -(-(cached[b] + new[b]) // bs))
            for j in range(held, want):
                tables[b, j] = free[taken] if taken < len(free) else -1
                taken += 1
    cu = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
    pos, slots = np.zeros(n_tokens, np.int64), np.full(n_tokens, -1, np.int64)
    for b in range(n):
        for i in range(new[b]):
            t, p = cu[b] + i, cached[b] + i
            if t < n_tokens:
                pos[t] = p
                if p // bs < w and tables[b, p // bs] >= 0:
                    slots[t] = int(tables[b, p // bs]) * bs + p % bs
    return tables, cu, pos, slots, np.add(new, cached), taken


def _check(gpu, new, cached, tables, bs, n_tokens, free, use_cached=True):
    t = torch.from_numpy(tables.copy()).to(gpu)
    f = None if free is None else _i32(free, gpu)
    m = paged.build_step_maps(_i32(new, gpu), _i32(cached, gpu) if use_cached else None, t, bs, n_tokens,
                              free_blocks=f)
    want = _host(new, cached, tables, bs, n_tokens, free)
    got = (t, m.cu_seqlens, m.positions, m.slot_mapping, m.context_lens)
    for g, w, name in zip(got, want, ("tables", "cu", "positions", "slots", "context")):
        assert np.array_equal(g.cpu().numpy(), w), name
    assert m.blocks_taken.tolist() == [want[5]]
    assert m.positions.dtype == m.slot_mapping.dtype == torch.int64
    return m


@pytest.mark.parametrize("n", [1, 3, 64, 65, 255, 256, 257, 1000])
@pytest.mark.parametrize("bs", [1, 16, 48, 256])
def test_random_steps(gpu, n, bs):
    print("case: maps", n, bs, flush=True)
    rs = np.random.RandomState(n * 1000 + bs)
    most = 40 if bs == 1 else 300
    new, cached = rs.randint(0, most, n), rs.randint(0, 2 * most, n)
    new[rs.rand(n) < 0.3] = 0
    w = int(((new + cached + bs - 1) // bs).max()) + 2
    held = (cached + bs - 1) // bs
    want = int(((new + cached + bs - 1) // bs - held).sum())
    ids = rs.permutation(int(held.sum()) + want + 3).astype(np.int32)
    tables = np.full((n, w), -7, np.int32)
    at = 0
    for b in range(n):
        tables[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    _check(gpu, new.tolist(), cached.tolist(), tables, bs, int(new.sum()), ids[at:].tolist())
    _check(gpu, new.tolist(), cached.tolist(), tables, bs, int(new.sum()) + 300, ids[at:].tolist())


def test_matches_the_host_metadata_of_a_prefill(gpu):
    lens = [1, 7, 300, 1024, 33]
    alloc = paged.BlockAllocator(40)
    alloc.allocate(3)
    free = list(alloc._free)
    blocks = [alloc.allocate(paged.blocks_needed(x, 64)) for x in lens]
    tables = paged.pad_block_tables(blocks, 17)
    cu, pos, slots = paged.build_prefill_metadata(lens, tables, 64, gpu, num_cache_rows=40 * 64)
    # complete tables
    t = torch.from_numpy(tables).to(gpu)
    m = paged.build_step_maps(_i32(lens, gpu), None, t, 64, sum(lens))
    assert torch.equal(m.cu_seqlens, cu) and torch.equal(m.positions, pos) and torch.equal(m.slot_mapping, slots)
    assert m.context_lens.tolist() == lens and m.blocks_taken.tolist() == [0]
    # tables filled from the free list
    t2 = torch.zeros_like(t)
    m = paged.build_step_maps(_i32(lens, gpu), None, t2, 64, sum(lens), free_blocks=_i32(free, gpu))
    assert torch.equal(t2, t) and torch.equal(m.slot_mapping, slots)
    assert m.blocks_taken.tolist() == [sum(map(len, blocks))]


def test_decode_steps_take_blocks_as_they_fill(gpu):
    """One token a sequence, step after step, the tables growing in place."""
    rs = np.random.RandomState(2)
    n, bs, w = 20, 16, 6
    cached = rs.randint(0, 40, n)
    held = (cached + bs - 1) // bs
    ids = rs.permutation(n * w).astype(np.int32)
    tables = np.full((n, w), -1, np.int32)
    at = 0
    for b in range(n):
        tables[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    t = torch.from_numpy(tables).to(gpu)
    ones = _i32([1] * n, gpu)
    lens = _i32(cached.tolist(), gpu)
    for _ in range(40):
        m = paged.build_step_maps(ones, lens, t, bs, n, free_blocks=_i32(ids[at:].tolist(), gpu))
        want = _host([1] * n, cached.tolist(), tables, bs, n, ids[at:].tolist())
        tables, cached = want[0], want[4]
        at += want[5]
        assert np.array_equal(t.cpu().numpy(), tables)
        assert np.array_equal(m.slot_mapping.cpu().numpy(), want[3])
        assert m.blocks_taken.tolist() == [want[5]]
        lens = m.context_lens


def test_exhausted_list_short_tables_and_cut_maps(gpu):
    tables = np.full((3, 4), -1, np.int32)
    new, cached = [40, 100, 20], [0, 0, 0]
    for free in ([], [5], [9, 8, 7, 6, 5]):
        _check(gpu, new, cached, tables, 16, 160, free)
    # positions past the table, negative lengths, fewer rows than tokens
    _check(gpu, [100, -4, 3], [0, 5, -9], tables, 16, 103, list(range(20)))
    _check(gpu, new, cached, tables, 16, 33, list(range(20)))
    _check(gpu, new, cached, tables, 16, 0, list(range(20)))
    _check(gpu, new, cached, tables, 16, 160, list(range(20)), use_cached=False)
    full = np.arange(12, dtype=np.int32).reshape(3, 4)
    full[1, 2] = -1
    _check(gpu, [30, 64, 1], [3, 0, 63], full, 16, 95, None)


def test_no_sequence(gpu):
    m = paged.build_step_maps(_i32([], gpu), None, torch.zeros((0, 4), dtype=torch.int32, device=gpu), 16, 5,
                              free_blocks=_i32([1], gpu))
    assert m.cu_seqlens.tolist() == [0] and m.slot_mapping.tolist() == [-1] * 5
    assert m.blocks_taken.tolist() == [0] and m.context_lens.numel() == 0


def test_most_sequences_and_one_more(gpu):
    n = paged.MAX_MAP_SEQS
    rs = np.random.RandomState(5)
    new, cached = rs.randint(0, 4, n), rs.randint(0, 50, n)
    tables = np.arange(n * 4, dtype=np.int32).reshape(n, 4)
    _check(gpu, new.tolist(), cached.tolist(), tables, 16, int(new.sum()), rs.permutation(n * 4).tolist())
    with pytest.raises(RuntimeError, match="at most"):
        paged.build_step_maps(_i32([1] * (n + 1), gpu), None,
                              torch.zeros((n + 1, 1), dtype=torch.int32, device=gpu), 16, 1)


def test_large_cache_rows(gpu):
    """Slots past 2^31."""
    tables = np.array([[2 ** 31 - 1, 2 ** 30]], np.int32)
    m = _check(gpu, [300], [200], tables, 256, 300, None)
    assert int(m.slot_mapping.max()) == (2 ** 31 - 1) * 256 + 255


def test_captured_and_replayed(gpu):
    rs = np.random.RandomState(6)
    n, bs, w = 30, 16, 12
    new, cached = _i32([0] * n, gpu), _i32([0] * n, gpu)
    t = torch.zeros((n, w), dtype=torch.int32, device=gpu)
    free = _i32(rs.permutation(n * w).tolist(), gpu)
    paged.build_step_maps(new, cached, t, bs, 2000, free_blocks=free)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m = paged.build_step_maps(new, cached, t, bs, 2000, free_blocks=free)
    for _ in range(3):
        a, c = rs.randint(0, 60, n), rs.randint(0, 100, n)
        new.copy_(_i32(a.tolist(), gpu))
        cached.copy_(_i32(c.tolist(), gpu))
        tables = rs.randint(0, n * w, (n, w)).astype(np.int32)
        t.copy_(torch.from_numpy(tables))
        g.replay()
        torch.cuda.synchronize()
        want = _host(a.tolist(), c.tolist(), tables, bs, 2000, free.tolist())
        assert np.array_equal(t.cpu().numpy(), want[0]) and np.array_equal(m.slot_mapping.cpu().numpy(), want[3])


def test_surface_refuses(gpu):
    l, t = _i32([1, 2], gpu), torch.zeros((2, 3), dtype=torch.int32, device=gpu)
    for a, o, match in [((l.long(), None, t, 16, 3), {}, "new_lens"), ((l, l[:1], t, 16, 3), {}, "cached"),
                        ((l, None, t[:1], 16, 3), {}, "block_tables"), ((l, None, t.long(), 16, 3), {}, "block_tables"),
                        ((l, None, t.t(), 16, 3), {}, "block_tables"), ((l, None, t, 0, 3), {}, "block_size"),
                        ((l, None, t, 16, -1), {}, "n_tokens"), ((l, None, t, 16, 3), dict(free_blocks=t), "free_blocks"),
                        ((l, None, t, 16, 3), dict(free_blocks=l.cpu()), "GPU")]:
        with pytest.raises(RuntimeError, match=match):
            paged.build_step_maps(*a, **o)
