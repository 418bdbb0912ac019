"""The plain definitions that the 4-bit pages and the page calls are held to, on their own (CPU)."""
import numpy as np
import pytest

import _pages_ref as ref


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("values", [False, True])
def test_pack_and_unpack(hd, values):
    """Values that are in the format come back, and others within half a step: d / 2 for the code, and the roundings of d, b and the
    value (2^-11 of 79 d, of |min| + 64 d, and of the value)."""
    rng = np.random.RandomState(hd + values)
    x = rng.randn(3, 2, 16, hd) * 1.3
    p = ref.pack(x, values)
    assert p.dtype == np.uint8 and p.shape == (3, 2, 16, 5 * hd // 8)
    y, d, b = ref.unpack(p, values)
    g = x.reshape(3, 2, 16, -1, 32)
    lo = g.min(-1, keepdims=True)
    bound = d[..., None] / 2 + 2.0 ** -11 * (79 * d[..., None] + np.abs(lo) + 64 * d[..., None] + np.abs(g))
    assert (np.abs(y.reshape(g.shape) - g) <= bound).all()
    n, d2, b2 = ref.quantise(x)
    assert np.array_equal(d2, d) and np.array_equal(b2, b)
    assert np.array_equal(y, ((64 + n.reshape(g.shape)) * d[..., None] + b[..., None]).astype(np.float16).reshape(x.shape))


def test_words_of_a_row():
    """The place of each code, by hand: row 5, element 8 w + 2 i in bits 4 i of word w, element 8 w + 2 i + 1 in bits 16 + 4 i."""
    x = np.zeros((1, 1, 16, 64))
    x[0, 0, 5, :] = np.arange(64) % 16
    for values in (False, True):
        words = ref.pack(x, values)[0, 0].reshape(-1)[:16 * 32].view(np.uint32)
        at = [((5 // 4) * 8 + w) * 4 + 5 % 4 if values else 5 * 8 + w for w in range(8)]
        assert [hex(v) for v in words[at]] == ["0x75316420", "0xfdb9eca8"] * 4
        assert words.sum() == words[at].sum()


def test_groups_that_have_no_pair():
    x = np.tile(np.linspace(-1, 1, 64), (1, 1, 16, 1))
    x[0, 0, 0, 3], x[0, 0, 1, 40], x[0, 0, 2, :32], x[0, 0, 3, 32:] = np.inf, np.nan, 7.0, np.linspace(-2e4, 2e4, 32)
    y, d, b = ref.unpack(ref.pack(x, False), False)
    nan = np.isnan(y[0, 0])
    assert nan[0, :32].all() and nan[1, 32:].all() and nan[3, 32:].all() and nan.sum() == 96
    assert (y[0, 0, 2, :32] == 7).all() and d[0, 0, 2, 0] == 0


def test_claims_one_after_another():
    """Three sequences that share a half-filled page and all write to it: the first two copy it, the last keeps it."""
    table = np.array([[0, 1, -1]] * 3, np.int32)
    refs = np.array([3, 3, 0, 0, 0], np.int32)
    new, counts, src, dst, lacking = ref.claim(table, refs, [0, 1, 2, 3], [25, 25, 25], 16)
    assert new.tolist() == [[0, 2, -1], [0, 3, -1], [0, 1, -1]] and counts.tolist() == [3, 1, 1, 1, 0]
    assert src.tolist() == [1, 1, -1] and dst.tolist() == [2, 3, -1] and lacking == 0
    new, counts, src, dst, lacking = ref.claim(table, refs, [0, 1, 2, 3], [33, 33, 33], 16)  # a new block each
    assert new.tolist() == [[0, 1, 2], [0, 1, 3], [0, 1, 4]] and (src == -1).all() and lacking == 0
    new, counts, src, dst, lacking = ref.claim(table, refs, [0, 20, 40, 60], [50, 50, 50], 16)  # blocks 1 (two copies) and 2
    assert lacking == 5 - 3 and (new == table).all() and (counts == refs).all()
