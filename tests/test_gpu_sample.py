"""dtts_sample_{f32,f16} against the definition in 64 bits: the same token, always, and its log-probability."""
import numpy as np
import pytest
import torch

from dtts import DttsError, serving

import _serving_ref as ref

pytestmark = pytest.mark.gpu
INF, LOWEST = float("inf"), float(np.finfo(np.float32).min)


def _run(dev, x, u, t=None, k=None, p=None, m=None, workspace=None):
    """x [rows, vocab] torch on the device, the rest lists; every row against the reference."""
    rows, vocab = x.shape

    def col(v, dtype):
        return None if v is None else torch.tensor(v, dtype=dtype, device=dev)

    f, i = torch.float32, torch.int32
    token, logprob = serving.sample(x, col(u, f), col(t, f), col(k, i), col(p, f), col(m, f), workspace)
    token, logprob = token.cpu().tolist(), logprob.cpu().double().tolist()
    xs = x.cpu().double().numpy()

    def at(v, r, d):
        return d if v is None else float(np.float32(v[r]))

    for r in range(rows):
        want, lp = ref.sample(xs[r], at(u, r, 0), at(t, r, 1.0), 0 if k is None else k[r], at(p, r, 1.0), at(m, r, 0.0))
        assert token[r] == want, (r, token[r], want, logprob[r], lp)
        # one f32 rounding, the weights' unit (half of 2^-42 a token of the sum), and x / T in f64
        tol = 2.0 ** -24 * abs(lp) + vocab * 2.0 ** -43 + 1e-12 if np.isfinite(lp) else 0.0
        assert logprob[r] == lp or abs(logprob[r] - lp) <= tol, (r, logprob[r], lp)
    return token


def _logits(dev, rows, vocab, dtype, seed, std=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g) * std).to(dtype).to(dev)


def _u(rows, seed):
    return torch.rand(rows, generator=torch.Generator().manual_seed(seed)).clamp(max=1 - 2.0 ** -24).tolist()


VOCABS = [1, 2, 63, 100, 257, 2048, 4096, 4097, 9001, 50021, 131072]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("vocab", VOCABS)
def test_sample_filters(dev, vocab, dtype):
    """Greedy, plain, each filter alone, all of them; f16 logits are full of ties."""
    rows = 12
    x = _logits(dev, rows, vocab, dtype, vocab)
    t = [0.0, 1.0, 0.7, 1.0, 0.9, 1.3, 0.05, 1.0, 5.0, 0.8, 1.0, 1.0]
    k = [0, 0, 1, 50, 0, 20, 40, 0, 400, vocab - 1, 10 ** 6, -3]
    p = [1.0, 1.0, 1.0, 1.0, 0.9, 0.8, 0.95, 1.0, 0.5, 1.0, 0.999, 1e-9]
    m = [0.0, 0.0, 0.0, 0.0, 0.0, 0.05, 0.0, 0.1, 0.0, 0.0, 0.5, 0.0]
    for seed in range(3):
        _run(dev, x, _u(rows, seed), t, k, p, m)
    _run(dev, x, _u(rows, 9))  # nothing given: plain sampling


@pytest.mark.parametrize("vocab", [7, 2048, 5000, 70001])
def test_sample_equal_logits(dev, vocab):
    """Every logit the same: top-k and top-p cut by index, u walks the whole range."""
    u = [0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 0.1]
    x = torch.full((6, vocab), -3.25, device=dev)
    _run(dev, x, u)
    got = _run(dev, x, u, k=[5] * 6)
    assert got == [0, 1, 2, 3, 4, 0]
    _run(dev, x, u, p=[0.5] * 6)
    _run(dev, x, u, k=[vocab // 2] * 6, p=[0.5] * 6, m=[1.0] * 6)
    # two levels: half of the tokens a little lower
    x[:, ::2] -= 1e-3
    _run(dev, x, u, k=[vocab * 3 // 4] * 6, p=[0.9] * 6)


@pytest.mark.parametrize("vocab", [2048, 40000])
def test_sample_narrow_and_wide_spreads(dev, vocab):
    """Logits within 1e-3 of each other (one histogram bin), and up to 1e4 apart (most of them weightless)."""
    base = _logits(dev, 4, vocab, torch.float32, 5, 1.0)
    for s in (1e-4, 1e3, 1e-30):
        _run(dev, base * s, _u(4, 6), [1.0, 0.3, 2.0, 1.0], [0, 100, vocab // 3, 1500], [0.7, 1.0, 0.9, 0.3])


@pytest.mark.parametrize("vocab", [300, 33000])
def test_sample_masked_rows(dev, vocab):
    """-inf, NaN and the lowest finite value in masked places; rows with one token left, none left, +inf."""
    x = _logits(dev, 9, vocab, torch.float32, 11)
    x[0, 100:] = -INF
    x[1, ::2] = float("nan")
    x[2, 5:] = LOWEST
    x[3, :] = -INF
    x[4, :] = float("nan")
    x[5, :] = -INF
    x[5, 37] = -4.0
    x[6, 20], x[6, 30] = INF, INF
    x[7, :] = LOWEST
    x[8, 250:] = -1e4
    for t in ([1.0] * 9, [0.0] * 9, [1e-30] * 9, [1e30] * 9, [INF] * 9):
        for k, p in (([0] * 9, [1.0] * 9), ([200] * 9, [0.9] * 9), ([3] * 9, [1.0] * 9), ([0] * 9, [0.7] * 9)):
            got = _run(dev, x, _u(9, 12), t, k, p)
            assert got[3] == -1 and got[4] == -1 and got[5] == 37
    _run(dev, x, [0.4] * 9, [1.0] * 9, [200] * 9, [0.9] * 9, [0.02] * 9)


def test_sample_odd_settings(dev):
    """Settings that are not numbers filter nothing (a temperature: greedy); u outside [0, 1) is clipped."""
    nan = float("nan")
    x = _logits(dev, 8, 500, torch.float32, 21)
    u = [nan, -1.0, 1.0, 2.0, INF, 0.5, 0.5, 0.5]
    _run(dev, x, u)
    _run(dev, x, u, t=[nan, -1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0], p=[1.0] * 5 + [nan, 0.0, -1.0], m=[0.0] * 5 + [nan, -1.0, 7.0])


def test_sample_zeros_of_both_signs_are_equal(dev):
    x = torch.full((2, 64), -9.0, device=dev)
    x[0, 10], x[0, 20] = -0.0, 0.0
    x[1, 10], x[1, 20] = 0.0, -0.0
    assert _run(dev, x, [0.0, 0.0], k=[1, 1]) == [10, 10]
    assert _run(dev, x, [0.9, 0.9], k=[2, 2]) == [20, 20]
    assert _run(dev, x, [0.9, 0.9], t=[0.0, 0.0]) == [10, 10]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("vocab", [1001, 20003])
def test_sample_strided_and_misaligned_rows(dev, vocab, dtype):
    wide = _logits(dev, 5, vocab + 9, dtype, 31)
    x = wide[:, 3:3 + vocab]
    _run(dev, x, _u(5, 32), [0.8] * 5, [60] * 5, [0.9] * 5)
    wide[:, :3], wide[:, 3 + vocab:] = 1000.0, 1000.0  # neighbours of the rows are none of theirs
    _run(dev, x, _u(5, 33), [0.8] * 5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_sample_largest_vocabulary(dev, dtype):
    vocab = 1 << 20
    x = _logits(dev, 3, vocab, dtype, 41)
    x[2] = 1.5
    _run(dev, x, [0.3, 0.99, 0.777], [1.0, 2.0, 1.0], [0, 5000, 0], [0.99, 0.9, 0.6])


def test_sample_many_rows(dev):
    rows = 3000
    x = _logits(dev, rows, 130, torch.float16, 51)
    _run(dev, x, _u(rows, 52), [0.9] * rows, [40] * rows, [0.9] * rows, [0.01] * rows)


def test_sample_follows_the_distribution(dev):
    """The u at the two ends of every token's share of the kept weight pick it and its neighbour."""
    x = _logits(dev, 1, 40, torch.float32, 61).expand(78, 40).contiguous()
    w = np.exp(x[0].cpu().double().numpy() - x[0].max().item())
    edge = np.cumsum(w)[:-1] / w.sum()
    u = np.stack([edge - 1e-6, edge + 1e-6], 1).ravel().astype(np.float32)
    got = serving.sample(x, torch.from_numpy(u).to(dev))[0].cpu().numpy().reshape(39, 2)
    assert np.array_equal(got, np.stack([np.arange(39), np.arange(1, 40)], 1))


@pytest.mark.parametrize("vocab", [500, 9000, 30000])
def test_sample_infinite_and_largest_logits(dev, vocab):
    """+inf takes all the weight from the largest finite number, at any temperature; equal weights at an infinite one."""
    x = _logits(dev, 4, vocab, torch.float32, 8)
    x[:2, 7], x[:2, vocab // 2], x[:2, vocab - 1] = INF, -LOWEST, INF
    x[3, 5:9] = -LOWEST
    for seed in range(3):
        u = _u(4, seed)
        for t in ([1.0, INF, INF, 1.0], [1e38, 1e-38, 1e38, INF]):
            got = _run(dev, x, u, t)
            assert got[0] in (7, vocab - 1) and got[1] in (7, vocab - 1)
            _run(dev, x, u, t, [0, 1, 9, 0], [0.5, 1.0, 0.9, 0.7], [0.0, 0.5, 0.1, 0.0])


@pytest.mark.parametrize("vocab", [1024, 1025, 2049, 8191, 8192, 8193, 10240, 16384, 16385])
def test_sample_where_the_kernel_changes(dev, vocab):
    """The last and first sizes of each row length's kernel; a min_p that nothing but the first token reaches."""
    x = _logits(dev, 6, vocab, torch.float32, vocab + 1)
    for seed in range(2):
        _run(dev, x, _u(6, seed), [1.0, 0.7, 1.0, 2.0, 1.0, 0.3], [0, 40, 0, vocab // 2, 0, 900], [1.0, 0.9, 0.7, 1.0, 1.0, 0.99],
             [0.0, 0.0, 0.0, 0.0, 1.5, 0.01])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("vocab", [9001, 16385, 131072])
def test_sample_without_a_workspace(dev, vocab, dtype):
    """One workgroup a row, or several: the same tokens and the same bits."""
    x = _logits(dev, 9, vocab, dtype, 3)
    x[8] = 1.0
    none = torch.empty(0, dtype=torch.uint8, device=dev)
    f, i = torch.float32, torch.int32
    t = torch.tensor([0.0, 1.0, 0.7, 1.0, 2.0, 0.1, 1.0, 1.0, 1.0], dtype=f, device=dev)
    k = torch.tensor([0, 0, 50, 0, 2000, vocab // 2, 0, 1, 300], dtype=i, device=dev)
    p = torch.tensor([1.0, 1.0, 0.9, 0.95, 0.5, 0.99, 1.0, 0.3, 0.5], dtype=f, device=dev)
    m = torch.tensor([0.0, 0.0, 0.0, 0.01, 0.0, 0.0, 0.2, 0.0, 0.0], dtype=f, device=dev)
    for seed in range(4):
        u = torch.tensor(_u(9, seed), dtype=f, device=dev)
        a, b = serving.sample(x, u, t, k, p, m), serving.sample(x, u, t, k, p, m, none)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_sample_refusals(dev):
    x = torch.zeros((2, 8), device=dev)
    u = torch.zeros(2, device=dev)
    with pytest.raises(DttsError, match="random numbers"):
        serving.sample(x, u[:1])
    with pytest.raises(DttsError, match="of top_k"):
        serving.sample(x, u, top_k=torch.zeros(3, dtype=torch.int32, device=dev))
    with pytest.raises(DttsError, match="top_k dtype"):
        serving.sample(x, u, top_k=torch.zeros(2, dtype=torch.int64, device=dev))
    with pytest.raises(DttsError, match="f32 or f16"):
        serving.sample(x.double(), u)
    with pytest.raises(DttsError, match="contiguous"):
        serving.sample(x.t(), torch.zeros(8, device=dev))
    with pytest.raises(DttsError, match="vocabulary"):
        serving.sample(torch.zeros((1, (1 << 20) + 1), device=dev), u[:1])
