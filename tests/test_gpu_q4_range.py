"""Attention over 4-bit pages where the weights of a row span many orders: a leading key over a long flat tail, and maxima that rise by
less than what moves a row's sums."""
import numpy as np
import pytest
import torch

from dtts import serving

import _pages_ref as pref

pytestmark = pytest.mark.gpu
PAGE = 64


def run(dev, scores, values, q_len, heads, n_kv, hd, workspace, window=0, sinks=0):
    """Attention of q_len tokens at the end of keys whose scores and values are one number each; and the 64-bit result of each token
    over what the pages stand for, with the mean of the values' magnitudes."""
    n = len(scores)
    pages = -(-n // PAGE)
    k, v = np.zeros((pages * PAGE, hd)), np.zeros((pages * PAGE, hd))
    k[:n, 3], v[:n] = scores, np.asarray(values)[:, None]
    packed = [pref.pack(np.ascontiguousarray(np.broadcast_to(t.reshape(pages, 1, PAGE, hd), (pages, n_kv, PAGE, hd))), i) for i, t in enumerate((k, v))]
    s, v = (pref.unpack(t[:, :1], i)[0].reshape(-1, hd)[:n, 3] for i, t in enumerate(packed))
    q = torch.zeros((q_len, heads, hd), dtype=torch.float16, device=dev)
    q[..., 3] = 1.0
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    table = torch.arange(pages, dtype=torch.int32, device=dev)[None].contiguous()
    ws = None if workspace else torch.empty(0, dtype=torch.uint8, device=dev)
    got = serving.paged_attention(q, *(torch.from_numpy(t).to(dev) for t in packed), i32([0, q_len]), i32([n]), table, q_len, n, 1.0,
                                  workspace=ws, window=window, sinks=sinks)
    want, mag = np.zeros(q_len), np.zeros(q_len)
    for i, p in enumerate(range(n - q_len, n)):
        j = np.arange(p + 1)
        j = j[(j > p - window) | (j < sinks)] if window else j
        w = np.exp(s[j] - s[j].max())
        want[i], mag[i] = (w * v[j]).sum() / w.sum(), (w * np.abs(v[j])).sum() / w.sum()
    return got.cpu().double().numpy().reshape(q_len, -1), want, mag


def check(got, want, mag, n):
    """Half a step of f16 in every weight and in the output (2^-11 each); f32: a lane adds at most n / 16 tiles' sums to its running
    ones, numerator and denominator (2^-24 each), a tile's sum has 32 terms, the exponent's argument (up to 64) is off by 2^-18; weights
    below f16's normal range by half of its smallest number (2^-25) under a largest weight of 2^11 at least."""
    rel = 2 * 2.0 ** -11 + (2 * n / 16 + 2 * 32) * 2.0 ** -24 + 2.0 ** -18
    tol = rel * mag + n * 2.0 ** -36 + 2.0 ** -25
    err = np.abs(got - want[:, None]).max(1)
    assert np.all(err <= tol), (float((err / tol).max()), got[-1, 0], want[-1])


SIZES = [(1, 1, 1, 128), (1, 8, 2, 64), (8, 4, 1, 128), (200, 4, 1, 128), (130, 1, 1, 64)]


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("q_len,heads,n_kv,hd", SIZES)
@pytest.mark.parametrize("below", [15.5, 17.5, 20.0])
def test_a_flat_tail_under_one_leading_key(dev, below, q_len, heads, n_kv, hd, workspace):
    """20001 keys; the leading one (value 0) first, inside, or last that every token sees."""
    n = 20001
    for at in (0, 9011, n - q_len):
        scores, values = np.full(n, -below), np.ones(n)
        scores[at], values[at] = 0.0, 0.0
        check(*run(dev, scores, values, q_len, heads, n_kv, hd, workspace), n)


@pytest.mark.parametrize("window,sinks", [(0, 0), (9000, 3)])
@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("q_len,heads,n_kv,hd", SIZES)
def test_a_maximum_that_rises_in_small_steps(dev, q_len, heads, n_kv, hd, workspace, window, sinks):
    """Leading keys 2.5 (under 2^4 in the weights) and 6 above the last: the rows keep an earlier one as their maximum, or move it."""
    n = 20003
    scores, values = np.full(n, -12.0), np.where(np.arange(n) % 2, 1.0, -0.5)
    for i, (at, s) in enumerate([(2, 0.0), (11500, 2.5), (13000, 8.5), (19000, 11.0)]):
        scores[at], values[at] = s, i - 1.5
    check(*run(dev, scores, values, q_len, heads, n_kv, hd, workspace, window, sinks), n)
