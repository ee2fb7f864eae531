"""Token log probabilities, entropy and top alternatives against float64 (oracle/kv4.py).

Bounds: S and T are float sums of at most 2^20 values in a tree (64 in a thread, six
shuffle steps, a few joins), each e^d with d rounded at 2^-24 |d| and the hardware's exp2
at one step: a relative error of S below 2^-17, of ln S the same absolutely; x - m is off by
half a step of it.  The entropy joins ln S and T / S (relative 2^-16)."""
import numpy as np
import pytest
import torch

from awesome_acceleration_amd import fused
from oracle import kv4 as oracle4
from gpu_util import f64

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _check(x, tokens, k, what=""):
    m = fused.token_logprobs(x, tokens, k)
    ref = f64(x)
    lp = oracle4.log_softmax(ref)
    t = tokens.cpu().numpy()
    want = np.array([0.0 if j < 0 else np.nan if j >= ref.shape[1] else lp[i, j] for i, j in enumerate(t)])
    ids = oracle4.top(ref, k)
    assert np.array_equal(m.top_ids.cpu().numpy(), ids), what
    for got, w in ((m.logprobs, want), (m.top_logprobs, np.take_along_axis(lp, ids, 1)),
                   (m.entropy, oracle4.entropy(ref))):
        g = f64(got)
        w = w.reshape(g.shape)
        fine = np.isfinite(w)
        assert np.array_equal(g[~fine], w[~fine], equal_nan=True), what
        assert (np.abs(g - w)[fine] <= 2.0 ** -16 * (1 + np.abs(w[fine]))).all(), what
    return m


def _rows(gpu, rs, rows, cols, dtype, size=3.0):
    return torch.from_numpy((rs.standard_normal((rows, cols)) * size).astype(np.float32)).to(DTYPES[dtype]).to(gpu)


def _tokens(gpu, rs, rows, cols):
    return torch.from_numpy(rs.randint(0, cols, rows)).to(gpu)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [1, 2, 7, 8, 9, 63, 64, 500, 2048, 16383, 16384, 16385, 32000, 50257, 151937])
def test_sizes(gpu, dtype, cols):
    print("case: logprobs", dtype, cols, flush=True)
    rs = np.random.RandomState(cols)
    x = _rows(gpu, rs, 3, cols, dtype)
    for k in {0, min(1, cols), min(5, cols), min(32, cols)}:
        _check(x, _tokens(gpu, rs, 3, cols), k, f"{cols} top {k}")


def test_largest_row(gpu):
    rs = np.random.RandomState(1)
    for dtype in ("bf16", "fp32"):
        x = _rows(gpu, rs, 2, 1 << 20, dtype)
        _check(x, _tokens(gpu, rs, 2, 1 << 20), 32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_misaligned_rows(gpu, dtype):
    rs = np.random.RandomState(2)
    wide = _rows(gpu, rs, 6, 5003, dtype)
    for a in range(4):
        x = wide[:, a:a + 4990]
        _check(x, _tokens(gpu, rs, 6, 4990), 6, f"offset {a}")
    _check(wide[1:2, 3:], _tokens(gpu, rs, 1, 5000), 6)
    x = wide[::2]
    _check(x, _tokens(gpu, rs, 3, 5003), 3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_take_the_lowest_index(gpu, dtype):
    rs = np.random.RandomState(3)
    x = torch.zeros((6, 40000), device=gpu, dtype=DTYPES[dtype])
    x[1] = -2.5
    x[2, 1::2] = 1.0                                     # half of the row
    x[3, torch.from_numpy(rs.permutation(40000)[:9]).to(gpu)] = 4.0
    x[4] = torch.from_numpy(rs.randint(-3, 4, 40000)).to(gpu)
    x[5, ::3] = -0.0
    for k in (1, 5, 32):
        _check(x, _tokens(gpu, rs, 6, 40000), k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sorted_rows(gpu, dtype):
    """The largest values in one wave's lanes, more than its list holds."""
    x = torch.arange(20000, device=gpu, dtype=torch.float32)
    x = torch.stack((x, -x, x % 700, -(x % 512))) / 1000
    _check(x.to(DTYPES[dtype]), torch.tensor([0, 19999, 3, 699], device=gpu), 32)
    _check(x.to(DTYPES[dtype]), torch.tensor([0, 19999, 3, 699], device=gpu), 2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_rows(gpu, dtype):
    """Fewer allowed tokens than alternatives; a row whose mask leaves nothing; the type's
    lowest value as the mask."""
    rs = np.random.RandomState(4)
    x = _rows(gpu, rs, 7, 33000, dtype)
    low = torch.finfo(x.dtype).min
    for r, (keep, value) in enumerate([(0, -np.inf), (1, -np.inf), (3, -np.inf), (100, -np.inf), (0, low), (2, low),
                                       (17000, -np.inf)]):
        mask = torch.ones(33000, dtype=torch.bool, device=gpu)
        mask[torch.from_numpy(rs.permutation(33000)[:keep]).to(gpu)] = False
        x[r, mask] = value
    for k in (0, 4, 20):
        _check(x, x.argmax(-1), k)
        _check(x, _tokens(gpu, rs, 7, 33000), k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_and_infinite_rows(gpu, dtype):
    rs = np.random.RandomState(5)
    x = _rows(gpu, rs, 5, 20000, dtype)
    x[0, 19999] = torch.nan
    x[1, 7] = torch.inf
    x[2, [3, 18000]] = torch.inf
    x[3, [5, 6, 17000]] = torch.nan
    x[3, 9] = torch.inf
    x[4, 0] = -torch.nan
    _check(x, _tokens(gpu, rs, 5, 20000), 6)


def test_large_logits(gpu):
    rs = np.random.RandomState(6)
    x = torch.from_numpy(rs.standard_normal((3, 9000)).astype(np.float32)).to(gpu)
    x[0] *= 1e4
    x[1] = x[1] * 1e-3 + 3e4
    x[2, 0], x[2, 1] = 3e38, -3e38
    _check(x, _tokens(gpu, rs, 3, 9000), 5)


def test_padding_and_out_of_range_tokens(gpu):
    rs = np.random.RandomState(7)
    x = _rows(gpu, rs, 4, 3000, "bf16")
    _check(x, torch.tensor([-1, 3000, -100, 2999], device=gpu), 2)


def test_agrees_with_argmax(gpu):
    rs = np.random.RandomState(8)
    x = _rows(gpu, rs, 50, 32000, "bf16")
    m = fused.token_logprobs(x, fused.argmax(x), 1)
    assert torch.equal(m.top_ids[:, 0], fused.argmax(x)) and torch.equal(m.top_logprobs[:, 0], m.logprobs)


def test_no_rows_and_refusals(gpu):
    x = torch.zeros((0, 10), device=gpu)
    m = fused.token_logprobs(x, torch.zeros(0, dtype=torch.int64, device=gpu), 3)
    assert m.logprobs.shape == (0,) and m.top_ids.shape == (0, 3)
    x, t = torch.zeros((3, 10), device=gpu), torch.zeros(3, dtype=torch.int64, device=gpu)
    for a, match in [((x[0], t, 1), "rows, cols"), ((x.t(), t, 1), "contiguous rows"), ((x.double(), t, 1), "dtype"),
                     ((x, t.int(), 1), "tokens"), ((x, t[:2], 1), "tokens"), ((x, t, 11), "top_k"), ((x, t, -1), "top_k"),
                     ((torch.zeros((3, 100), device=gpu), t, 33), "top_k"), ((x[:1].expand(3, 10), t, 1), "overlap")]:
        with pytest.raises(RuntimeError, match=match):
            fused.token_logprobs(*a)


def test_captured_replayed_and_on_another_stream(gpu):
    rs = np.random.RandomState(9)
    x, t = _rows(gpu, rs, 5, 70001, "bf16"), _tokens(gpu, rs, 5, 70001)
    fused.token_logprobs(x, t, 7)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m = fused.token_logprobs(x, t, 7)
    side = torch.cuda.Stream()
    for _ in range(3):
        x.normal_()
        eager = fused.token_logprobs(x, t, 7)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = fused.token_logprobs(x, t, 7)
        g.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(m, eager, other):
            assert torch.equal(a, b) and torch.equal(c, b)
    _check(x, t, 7)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_about_the_most_groups_read_whole(gpu, dtype):
    """Columns about 64 and 128 groups of maxima, from every place of a 16-byte boundary on,
    and values whose largest lie in one group or in every one."""
    rs = np.random.RandomState(30)
    group = 64 if dtype == "fp32" else 128
    for cols in (64 * group, 128 * group):
        for off in (0, 1, 3, 7):
            n = cols + int(rs.randint(-9, 10))
            wide = _rows(gpu, rs, 3, n + 16, dtype)
            x = wide[:, off:off + n]
            x[1, 700:732] += 30.0                 # the top within one group and its neighbour
            x[2, ::group] += 30.0                 # a large one in each
            for k in (1, 20, 32):
                _check(x, _tokens(gpu, rs, 3, n), k, f"{n} columns from {off}, top {k}")
