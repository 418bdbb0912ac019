"""dtts_paged_attention_f16 where the weights of a row span many orders: one or two keys ahead of a long flat tail, whose
weights are each next to nothing and together are not."""
import numpy as np
import pytest
import torch

from dtts import serving

pytestmark = pytest.mark.gpu
PAGE = 64


def _run(dev, scores, values, q_len, heads, n_kv, hd, workspace):
    """Attention of q_len tokens at the end of keys whose scores (exact in f16) and values are one number each, for every
    token alike; the 64-bit result of each token."""
    n = len(scores)
    pages = -(-n // PAGE)
    s, v = np.zeros(pages * PAGE), np.full(pages * PAGE, np.nan)
    s[:n], v[:n] = scores, values
    k = torch.zeros((pages, n_kv, PAGE, hd), dtype=torch.float16)
    k[..., 3] = torch.from_numpy(s).half().view(pages, 1, PAGE)
    vv = torch.from_numpy(v).half().view(pages, 1, PAGE, 1).expand(pages, n_kv, PAGE, hd).contiguous()
    assert np.array_equal(k[:, 0, :, 3].double().numpy().ravel(), s)
    q = torch.zeros((q_len, heads, hd), dtype=torch.float16, device=dev)
    q[..., 3] = 1.0
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    table = torch.arange(pages, dtype=torch.int32, device=dev)[None].contiguous()
    ws = None if workspace else torch.empty(0, dtype=torch.uint8, device=dev)
    got = serving.paged_attention(q, k.to(dev), vv.to(dev), i32([0, q_len]), i32([n]), table, q_len, n, 1.0, workspace=ws)
    w = np.exp(s[:n] - s[:n].max())
    v = vv[:, 0, :, 0].double().numpy().ravel()[:n]
    num, den, mag = (np.cumsum(x)[n - q_len:] for x in (w * v, w, w * np.abs(v)))
    return got.cpu().double().numpy().reshape(q_len, -1), num / den, mag / den


def _check(got, want, mag, n, small):
    """Half a step of f16 in every weight and in the output (2^-11 each); f32: a lane adds at most n / 16 products' or tiles'
    sums to its running ones, numerator and denominator (2^-24 each), a tile's sum has 32 terms, the exponent's argument (up
    to 64) is off by 2^-18; weights below f16's normal range by at most `small` of the largest each."""
    rel = 2 * 2.0 ** -11 + (2 * n / 16 + 2 * 32) * 2.0 ** -24 + 2.0 ** -18
    tol = rel * mag + n * small + 2.0 ** -25
    err = np.abs(got - want[:, None]).max(1)
    assert np.all(err <= tol), (float((err / tol).max()), got[-1, 0], want[-1])


# half of f16's smallest number (2^-25) under a largest weight of 2^15 (16-row tiles) and of 2^11 at least (128-row ones)
SMALL = {True: 2.0 ** -40, False: 2.0 ** -36}


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("q_len,heads,n_kv,hd", [(1, 1, 1, 128), (1, 8, 2, 64), (8, 4, 1, 128), (200, 4, 1, 128), (130, 1, 1, 64)])
@pytest.mark.parametrize("below", [15.5, 17.0, 17.5, 20.0])
def test_a_flat_tail_under_one_leading_key(dev, below, q_len, heads, n_kv, hd, workspace):
    """65001 keys; the leading one (value 0) first, inside, or last that every token sees."""
    n = 65001
    for at in (0, 30011, n - q_len):
        scores, values = np.full(n, -below), np.ones(n)
        scores[at], values[at] = 0.0, 0.0
        got, want, mag = _run(dev, scores, values, q_len, heads, n_kv, hd, workspace)
        _check(got, want, mag, n, SMALL[q_len * heads // n_kv <= 32])


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("q_len,heads", [(1, 4), (200, 4)])
def test_a_maximum_that_rises_in_small_steps(dev, q_len, heads, workspace):
    """Leading keys 2.5 (under 2^4 in the weights) and 6 above the last: the 128-row tiles keep an earlier one as their
    maximum, or move it."""
    n = 30003
    scores, values = np.full(n, -12.0), np.where(np.arange(n) % 2, 1.0, -0.5)
    for i, (at, s) in enumerate([(2, 0.0), (500, 2.5), (9000, 8.5), (20000, 11.0)]):
        scores[at], values[at] = s, i - 1.5
    got, want, mag = _run(dev, scores, values, q_len, heads, 1, 128, workspace)
    _check(got, want, mag, n, SMALL[q_len * heads <= 32])


@pytest.mark.parametrize("hd,heads", [(64, 1), (64, 8), (128, 1), (128, 8)])
@pytest.mark.parametrize("n", [33000, 65000])
def test_a_row_of_hundreds_of_chunks(dev, n, hd, heads):
    """One token of one kv head is cut into more than 256 chunks, which its join takes in several rounds: with the largest
    score in the first round, in the last one and in the chunk between them, the rest rising or falling."""
    assert serving.paged_attention_workspace_bytes(1, 1, heads, 1, hd, 1, n) > 256 * heads * (hd + 4) * 4
    rng = np.random.RandomState(n + hd)
    values = rng.randint(-8, 9, n) / 4.0
    for at in (5, n // 2, n - 3):
        for slope in (0.0, 6.0, -6.0):
            scores = np.round((rng.rand(n) * 2 + slope * np.arange(n) / n) * 64) / 64
            scores[at] = 12.0
            got, want, mag = _run(dev, scores, values, 1, heads, 1, hd, True)
            _check(got, want, mag, n, SMALL[True])


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("q_len,heads,n_kv,hd,n", [(1, 2, 1, 128, 300), (7, 4, 2, 64, 900), (100, 2, 1, 128, 300), (200, 2, 2, 64, 1200)])
@pytest.mark.parametrize("scale", [0.3, 1.0, 30.0, -30.0, 1e3, 1e9, 1e20, -1e32, 2e38])
def test_scores_of_any_size(dev, scale, q_len, heads, n_kv, hd, n, workspace):
    """Scores of whole numbers times 2^9 times the scale, up to past f32's range: a token has the value of its largest one, or
    the mean of those that share it."""
    rng = np.random.RandomState(7)
    pages = -(-n // PAGE)
    # q . k = 2^9 (64 a + b), a and b whole: exact in f32, and any two are equal or 2^9 apart at least
    a, b = rng.randint(-500, 501, (pages * PAGE, n_kv)), rng.randint(-200, 201, (pages * PAGE, n_kv))
    if n == 900:
        b[:] = 0  # many keys share a score
        a = a // 100 * 100
    k = torch.zeros((pages * PAGE, n_kv, hd), dtype=torch.float16)
    k[:, :, 5], k[:, :, hd - 1] = torch.from_numpy(a).half(), torch.from_numpy(b).half()
    v = torch.randn((pages * PAGE, n_kv, hd), generator=torch.Generator().manual_seed(5)).half()
    paged = [t.view(pages, PAGE, n_kv, hd).transpose(1, 2).contiguous().to(dev) for t in (k, v)]
    q = torch.zeros((q_len, heads, hd), dtype=torch.float16, device=dev)
    q[..., 5], q[..., hd - 1] = 2.0 ** 15, 2.0 ** 9
    score = (64 * a + b).astype(np.int64)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    ws = None if workspace else torch.empty(0, dtype=torch.uint8, device=dev)
    got = serving.paged_attention(q, *paged, i32([0, q_len]), i32([n]), torch.arange(pages, dtype=torch.int32, device=dev)[None].contiguous(),
                                  q_len, n, scale, workspace=ws).cpu().double()
    for t in range(q_len):
        for h in range(heads):
            s = score[:n - q_len + t + 1, h // (heads // n_kv)] * (1 if scale > 0 else -1)
            best = torch.from_numpy(np.flatnonzero(s == s.max()))
            x = v[best, h // (heads // n_kv)].double()
            # the next score is 2^9 times 0.3 below at least: its weight is under e^-150 of the largest. f16: equal weights round
            # alike (numerator 2^-11 against the unrounded sum), the output 2^-11; a few f32 steps
            tol = (2 * 2.0 ** -11 + 2.0 ** -18) * x.abs().mean(0) + 2.0 ** -25
            assert bool(((got[t, h] - x.mean(0)).abs() <= tol).all()), (t, h, len(best), float((got[t, h] - x.mean(0)).abs().max()))


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("q_len,heads,n_kv,hd,n", [(1, 2, 1, 128, 200), (1, 8, 2, 64, 3000), (8, 4, 2, 64, 900), (100, 2, 2, 128, 300), (200, 4, 1, 64, 1500)])
@pytest.mark.parametrize("base", [2.0 ** 10, 2.0 ** 13, 2.0 ** 18, 2.0 ** 20, -2.0 ** 20])
def test_large_scores_that_differ_by_little(dev, base, q_len, heads, n_kv, hd, n, workspace):
    """Scores of `base` and up to 8 more, in quarters (exact in f32): their differences count in full, also between the keys
    of several waves, tiles and chunks."""
    rng = np.random.RandomState(int(abs(base)) % 97 + n)
    pages = -(-n // PAGE)
    more = rng.randint(0, 33, (pages * PAGE, n_kv)) / 4.0
    k = torch.zeros((pages * PAGE, n_kv, hd), dtype=torch.float16)
    k[:, :, 5], k[:, :, hd - 1] = base / 2.0 ** 10, torch.from_numpy(more).half()
    v = torch.randn((pages * PAGE, n_kv, hd), generator=torch.Generator().manual_seed(5)).half()
    paged = [t.view(pages, PAGE, n_kv, hd).transpose(1, 2).contiguous().to(dev) for t in (k, v)]
    q = torch.zeros((q_len, heads, hd), dtype=torch.float16, device=dev)
    q[..., 5], q[..., hd - 1] = 2.0 ** 10, 1.0
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    ws = None if workspace else torch.empty(0, dtype=torch.uint8, device=dev)
    got = serving.paged_attention(q, *paged, i32([0, q_len]), i32([n]), torch.arange(pages, dtype=torch.int32, device=dev)[None].contiguous(),
                                  q_len, n, 1.0, workspace=ws).cpu().double()
    w = torch.from_numpy(np.exp(more - 8.0))[:, :, None]
    x = v.double()
    num, den, mag = ((w * x).cumsum(0), w.cumsum(0), (w * x.abs()).cumsum(0))
    rows = slice(n - q_len, n)
    want, mag = (num[rows] / den[rows]), (mag[rows] / den[rows])
    got = got.view(q_len, n_kv, heads // n_kv, hd)
    # f16: 2^-11 of each weight and of the output; a maximum's rounded product: 2^-13 in base 2 where it is under 2^12, twice
    # (what was summed and what it joins); f32: the sums, the scale's own rounding (2^-24 of a difference up to 8 * 1.45)
    tol = (2 * 2.0 ** -11 + 2 * 2.0 ** -13 * 0.7 + (2 * n / 16 + 64) * 2.0 ** -24 + 2.0 ** -19) * mag + 2.0 ** -25
    err = (got - want[:, :, None]).abs()
    assert bool((err <= tol[:, :, None]).all()), float((err / tol[:, :, None]).max())
