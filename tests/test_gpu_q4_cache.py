"""The 4-bit cache: the append that writes it, its values read back, and attention over it, against 64-bit evaluations."""
import numpy as np
import pytest
import torch

from dtts import DttsError, serving

import _pages_ref as pref
import _serving_ref as ref

pytestmark = pytest.mark.gpu

NAMES = ("rotary", "qk_rope_append_paged", "paged_attention", "sample", "unpack_pages")


@pytest.fixture(params=["binding", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        for name in NAMES:
            monkeypatch.setattr(serving._serving, name, lambda *args: None)


def q4(b, stride_pages=1):
    """A _serving_ref.Batch's pages in 4 bits: (k, v, the f16 values they stand for); slots that hold no position are NaN."""
    packed = [pref.repack(t, i, stride_pages) for i, t in enumerate((b.k, b.v))]
    values = [torch.from_numpy(pref.unpack(t.contiguous().numpy(), i)[0]).half() for i, t in enumerate(packed)]
    return [torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=b.dev).copy_(t) for t in packed], values


def tables(dev, length, rot):
    return (torch.from_numpy(t).to(dev) for t in serving.rope_table_scaled(length, rot, 1e4))


# ---------------------------------------------------------------- unpack

@pytest.mark.parametrize("hd,page,n_kv,stride", [(64, 16, 1, 1), (64, 64, 3, 2), (128, 16, 2, 1), (128, 32, 5, 3), (64, 256, 1, 1)])
def test_unpack(dev, path, hd, page, n_kv, stride):
    """Any bytes: codes and pairs of all kinds, infinities, NaN and subnormal ones among them, bit for bit."""
    rng = np.random.RandomState(hd + page)
    raw = [rng.randint(0, 256, (7, n_kv, page, 5 * hd // 8)).astype(np.uint8) for _ in range(2)]
    want = [pref.unpack(t, i)[0].astype(np.float16) for i, t in enumerate(raw)]
    wide = [torch.zeros((7 * stride, *t.shape[1:]), dtype=torch.uint8, device=dev)[::stride].copy_(torch.from_numpy(t)) for t in raw]
    for got, w in zip(serving.unpack_pages(*wide), want):
        got = got.cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(w)) and np.array_equal(got[~np.isnan(w)], w[~np.isnan(w)])
    ids = torch.tensor([6, 2, 2, -1, 7, 0], dtype=torch.int32, device=dev)
    for got, w in zip(serving.unpack_pages(*wide, ids), want):
        got, w = got.cpu().numpy()[[0, 1, 2, 5]], w[[6, 2, 2, 0]]
        assert got.shape == w.shape and np.array_equal(got[~np.isnan(w)], w[~np.isnan(w)])
    assert serving.unpack_pages(*wide, ids[:0])[0].shape == (0, n_kv, page, hd)


# ---------------------------------------------------------------- append

@pytest.mark.parametrize("hd,rot,interleaved", [(128, 128, False), (128, 64, False), (128, 40, False), (128, 128, True), (64, 64, False),
                                                (64, 8, False), (64, 16, True), (64, 56, False)])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("norm", [False, True])
def test_append(dev, path, hd, rot, interleaved, dtype, norm):
    """Values within what their codes allow: with d = (max - min) / 15 of the exact row, half a step and what the roundings move
    the ends by: those of d, b and the value in f16 (2^-11 each of 79 d, |min| + 64 d, |x|), and those of the row's norm and
    rotation in f32 (under 2^-18 of its largest). Slots of no new token keep their bits."""
    heads, n_kv, page = 5, 3, 16
    b = ref.Batch([1, 0, 5, 33, 1], [7, 20, 5, 80, 64], n_kv, hd, page, dev, seed=hd + rot, extra_tokens=2)
    (k, v), _ = q4(b)
    before = [t.cpu().numpy() for t in (k, v)]
    _, _, start, ctx, table = b.device()
    g = torch.Generator().manual_seed(rot)
    x = torch.randn((b.tokens, (heads + 2 * n_kv) * hd), generator=g)
    x = x.half() if dtype == "f16" else x
    norms = torch.rand((2, hd), generator=g) + 0.5 if norm else None
    cos, sin = tables(dev, 128, rot)
    q = serving.qk_rope_append_paged(x.to(dev), cos, sin, k, v, start, ctx, table, heads, norms=None if norms is None else norms.to(dev),
                                     eps=1e-6, interleaved=interleaved, out=torch.full((b.tokens, heads, hd), 9.0, device=dev).half())
    seq = np.repeat(np.arange(5), b.n)
    pos = np.concatenate([np.arange(c - n, c) for n, c in zip(b.n, b.c)])
    t = int(b.start[-1])
    rows = x.double().numpy().reshape(b.tokens, -1, hd)[:t]
    qr, kr, vr = rows[:, :heads], rows[:, heads:heads + n_kv], rows[:, heads + n_kv:]
    if norm:
        w = norms.double().numpy()
        qr, kr = ref.rms(qr, w[0], 1e-6), ref.rms(kr, w[1], 1e-6)
    c, s = (a.cpu().double().numpy()[pos] for a in (cos, sin))
    (qr, qm), (kr, _) = ref.turn(qr, c, s, interleaved), ref.turn(kr, c, s, interleaved)
    assert (np.abs(q[:t].cpu().double().numpy() - qr) <= 2.0 ** -11 * np.abs(qr) + 2.0 ** -20 * qm + 2.0 ** -25).all()
    assert bool((q[t:] == 9.0).all())
    for i, (pages, want, old) in enumerate(zip((k, v), (kr, vr), before)):
        raw = pages.cpu().numpy()
        got, d, base = pref.unpack(raw, i)
        at = b.table[seq, pos // page], slice(None), pos % page
        y, w = got[at].reshape(t, n_kv, -1, 32), want.reshape(t, n_kv, -1, 32)
        lo = w.min(-1, keepdims=True)
        step = (w.max(-1, keepdims=True) - lo) / 15
        bound = step / 2 + 2.0 ** -11 * (79 * step + np.abs(lo) + 64 * step + np.abs(w)) + 2.0 ** -18 * np.abs(want).max(-1)[..., None, None]
        assert (np.abs(y - w) <= bound).all(), np.max(np.abs(y - w) / bound)
        assert (np.abs(d[at][..., None] - step) <= 2.0 ** -11 * step + 2.0 ** -18 * np.abs(want).max(-1)[..., None, None]).all()
        # the other slots: their codes and pairs, all bits (as values NaN hides them)
        kept = np.ones((len(raw), page), bool)
        kept[at[0], at[2]] = False
        for x0, x1 in zip(slots(old, i), slots(raw, i)):
            assert np.array_equal(x0[kept], x1[kept])


def test_append_of_f16_values_takes_the_codes_of_the_definition(dev):
    """Values of f16 rows go into their pages without arithmetic before it, so their codes and pairs are the definition's, ties
    between two codes (which the f16 grid has many of) included."""
    n_kv, page = 2, 64
    for hd in (64, 128):
        x = (torch.randn((page, (1 + 2 * n_kv) * hd), generator=torch.Generator().manual_seed(hd)) * 2).half()
        x[:, -hd:] = (x[:, -hd:] * 8).round() / 8  # a coarse grid: a tie every few values
        cos, sin = tables(dev, page, hd)
        k, v = (torch.zeros((1, n_kv, page, 5 * hd // 8), dtype=torch.uint8, device=dev) for _ in range(2))
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
        serving.qk_rope_append_paged(x.to(dev), cos, sin, k, v, i32([0, page]), i32([page]), i32([[0]]), 1)
        want = pref.pack(x[:, -n_kv * hd:].double().numpy().reshape(page, n_kv, hd).transpose(1, 0, 2)[None], True)
        assert np.array_equal(v.cpu().numpy(), want), hd


def hard_groups(rng, n):
    """Groups [5 n, 32] of f32 numbers: whose width over 15, and whose least number less 64 steps, are next to half way between two
    f16 numbers, nearer than f32 can tell; narrow ones far from zero, whose first code is no f32 number; ones whose least number is 64
    steps and next to nothing; ordinary ones."""
    f = np.float32
    d = rng.randint(1024, 2048, n) * 2.0 ** rng.randint(-13, -3, n)
    sign = rng.choice([-1, 1], n)
    mid = rng.rand(n, 32)

    def ends(lo, hi):
        g = (lo[:, None] + mid * (hi - lo)[:, None]).astype(f)
        g = g.clip(lo.astype(f)[:, None], hi.astype(f)[:, None])
        g[:, 3], g[:, 7] = lo, hi
        return g

    tie = 15 * (d + 2.0 ** (np.floor(np.log2(d)) - 11))
    low = sign * tie * 2.0 ** -26
    least = (-64 * d * (1 + rng.uniform(-0.02, 0.02, n))).astype(np.float16)
    half = np.spacing(np.abs(least)).astype(np.float64) / 2
    lo = np.nextafter((least.astype(np.float64) + half + 64 * d).astype(f), (sign * 1e9).astype(f)).astype(np.float64)
    at = sign * 10 ** rng.uniform(-2, 3.3, n)
    near = 64 * d + sign * 2.0 ** rng.uniform(-24, -10, n)
    return np.concatenate([ends(low, tie), ends(lo, lo + 15 * d), ends(at, at + 10 ** rng.uniform(-5, -1, n)),
                           ends(near, near + 15 * d), rng.randn(n, 32).astype(f)])


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_of_f32_values_takes_the_pairs_and_codes_of_the_definition(dev, interleaved):
    """Rows that the rotation leaves as they are: pairs bit for bit, codes but for those of values within 2^-18 of a step of the border
    between two (three f32 roundings of 16 steps at most)."""
    n_kv, page, hd = 4, 64, 128
    rng = np.random.RandomState(5)
    g = rng.permutation(hard_groups(rng, page * n_kv * 2))[:page * n_kv * 8]
    rows = torch.from_numpy(g.reshape(page, 2 * n_kv, hd))
    x = torch.cat([torch.zeros((page, 1, hd)), rows], 1).view(page, -1)
    cos, sin = torch.ones((page, hd // 2), device=dev), torch.zeros((page, hd // 2), device=dev)
    pages = [torch.zeros((1, n_kv, page, 80), dtype=torch.uint8, device=dev) for _ in range(2)]
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    serving.qk_rope_append_paged(x.to(dev), cos, sin, *pages, i32([0, page]), i32([page]), i32([[0]]), 1, interleaved=interleaved)
    for i, t in enumerate(pages):
        want = rows[:, i * n_kv:(i + 1) * n_kv].double().numpy()  # [page, n_kv, D]
        n, d, b = pref.quantise(want)
        words, pairs = slots(t.cpu().numpy(), i)
        pairs = np.ascontiguousarray(pairs[0]).view(np.float16).reshape(page, n_kv, hd // 32, 2)
        assert np.array_equal(pairs[..., 0].view(np.int16), d.view(np.int16)) and np.array_equal(pairs[..., 1].view(np.int16), b.view(np.int16))
        got = np.stack([words[0] >> np.uint32(4 * (e // 2) + 16 * (e % 2)) & np.uint32(15) for e in range(8)], -1).reshape(want.shape)
        d, b = (np.repeat(y.astype(np.float64), 32, -1) for y in (d, b))
        step = (want.astype(np.longdouble) - b - 64 * d) / np.where(d > 0, d, 1)
        border = np.abs(step - np.floor(step) - 0.5)
        assert (border[got != n] <= 2.0 ** -18).all(), (got != n).sum()


def slots(raw, values):
    """The words [n_pages, page, n_kv, D / 8] and pairs [n_pages, page, n_kv, D / 32] of uint8 pages."""
    n, n_kv, page, row = raw.shape
    hd = row * 8 // 5
    flat = np.ascontiguousarray(raw.reshape(n, n_kv, -1)).view(np.uint32)
    w = flat[..., :page * hd // 8]
    w = w.reshape(n, n_kv, page // 4, hd // 8, 4).swapaxes(-1, -2) if values else w
    return w.reshape(n, n_kv, page, hd // 8).swapaxes(1, 2), flat[..., page * hd // 8:].reshape(n, n_kv, hd // 32, page).transpose(0, 3, 1, 2)


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_of_values_that_have_no_pair(dev, interleaved):
    """A group with an infinity or a NaN, or too wide for f16's range, is NaN and no other; a flat one is its value; zeros are zeros.
    Rows at position 0, whose rotation leaves what is finite as it is."""
    hd = 128
    x = torch.randn((6, 3 * hd), generator=torch.Generator().manual_seed(3))
    x[0, hd + 5], x[1, hd + 40], x[2, 2 * hd + 100] = float("inf"), float("nan"), -float("inf")
    x[3, hd:hd + 32], x[3, 2 * hd:] = 0.3, 0.0
    x[4, 2 * hd:2 * hd + 32] = torch.linspace(-20000, 20000, 32)
    x[5, hd:2 * hd], x[5, 2 * hd:] = torch.linspace(0, 1e-6, hd), torch.linspace(60000, 65000, hd)
    cos, sin = tables(dev, 16, hd)
    k, v = (torch.full((6, 1, 16, 80), 7, dtype=torch.uint8, device=dev) for _ in range(2))
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    serving.qk_rope_append_paged(x.to(dev), cos, sin, k, v, i32(range(7)), i32([1] * 6), i32([[i] for i in range(6)]), 1,
                                 interleaved=interleaved)
    k, v = (pref.unpack(t.cpu().numpy(), i)[0][:, 0, 0] for i, t in enumerate((k, v)))
    nan = np.zeros((2, 6, 4), bool)
    nan[0, 0, 0] = nan[0, 1, 1] = nan[1, 2, 3] = nan[1, 4, 0] = True
    if not interleaved:  # x2 + x1 sin 0 of a key's pair half a row away: 0 times what is not finite
        nan[0, 0, 2] = nan[0, 1, 3] = True
    got = np.isnan(np.stack([k, v])).reshape(2, 6, 4, 32)
    assert bool((got == nan[..., None]).all()), np.argwhere(got != nan[..., None])[:5]
    assert (k[3, :32] == np.float16(0.3)).all() and (v[3] == 0).all()
    # wide means: a step is f16's where its width is less (2^-24 apart under 2^-14, 32 apart at 60000)
    assert (np.abs(k[5] - x[5, hd:2 * hd].numpy()) <= 1e-6 / 4 / 15 / 2 + 3 * 2.0 ** -25 + 64 * 2.0 ** -25).all()
    assert (np.abs(v[5] - x[5, 2 * hd:].numpy()) <= 1250 / 15 / 2 + 2.0 ** -11 * (65000 * 2 + 143 * 1250 / 15)).all()


# ---------------------------------------------------------------- attention

def check(b, packed, values, q, max_q, max_context, scale, window=0, sinks=0, workspace=None):
    _, _, start, ctx, table = b.device()
    q = q.to(b.dev)
    out = torch.full((b.tokens, q.shape[1], b.hd), 9.0, dtype=torch.float16, device=b.dev)
    got = serving.paged_attention(q, *packed, start, ctx, table, max_q, max_context, scale, window, out=out, sinks=sinks, workspace=workspace)
    t = int(b.start[-1])
    want, bound = pref.attention(q, *values, b.start, b.c, b.table, b.page, scale, window, sinks)
    err = (got[:t].cpu().double() - want[:t]).abs()
    assert bool((err <= bound[:t]).all()), f"{(err / bound[:t]).max()} of the bound"
    assert bool((got[t:] == 9.0).all())
    return got


SHAPES = [  # n, context, n_kv, gqa, D, page
    ([1], [1], 1, 1, 128, 16), ([1], [33], 2, 2, 64, 16), ([1, 1, 1], [300, 17, 64], 2, 8, 128, 16), ([1, 0, 2], [65, 9, 130], 1, 5, 64, 64),
    ([7], [7], 1, 4, 128, 32), ([40], [161], 2, 1, 64, 16), ([33, 1, 5], [250, 250, 5], 1, 4, 128, 128), ([70, 30], [70, 400], 2, 2, 128, 16),
    ([129], [300], 1, 3, 64, 32), ([1], [1500], 1, 1, 128, 16), ([2] * 17, [90 + 7 * i for i in range(17)], 1, 2, 128, 16),
]


@pytest.mark.parametrize("n,c,n_kv,gqa,hd,page", SHAPES)
def test_attention(dev, path, n, c, n_kv, gqa, hd, page):
    b = ref.Batch(n, c, n_kv, hd, page, dev, seed=len(n) + hd, extra_tokens=1)
    packed, values = q4(b)
    q = (torch.randn((b.tokens, n_kv * gqa, hd), generator=torch.Generator().manual_seed(hd)) * 1.3).half()
    for max_q, workspace in ((max(n), None), (max(n), torch.empty(0, dtype=torch.uint8, device=dev)), (1, None), (500, None)):
        check(b, packed, values, q, max_q, max(c), hd ** -0.5, workspace=workspace)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (40, 3), (64, 64), (100, 65), (33, 500), (1000, 4), (16, 200)])
@pytest.mark.parametrize("n,c,hd", [([1, 1], [300, 40], 64), ([1, 3, 50], [700, 140, 333], 128), ([90], [450], 64), ([40], [900], 128)])
def test_attention_with_windows_and_sinks(dev, window, sinks, n, c, hd):
    b = ref.Batch(n, c, 2, hd, 16, dev, seed=window, extra_tokens=1)
    packed, values = q4(b)
    q = torch.randn((b.tokens, 4, hd), generator=torch.Generator().manual_seed(hd)).half()
    for max_q in (max(n), 1):
        check(b, packed, values, q, max_q, max(c), -0.2, window, sinks)


def test_attention_rows_and_pages_apart(dev, path):
    """Queries inside wider rows, pages with others between them, pages that are not there."""
    b = ref.Batch([1, 30, 1], [100, 90, 40], 2, 128, 16, dev, seed=5)
    b.table[0, 2] = b.table[1, 0] = -1
    b.table[2, 1] = b.n_pages
    packed, values = q4(b, 3)
    assert packed[0].stride(0) == 3 * 2 * 16 * 80
    wide = torch.randn((b.tokens, 9, 128), generator=torch.Generator().manual_seed(1)).half().to(dev)
    check(b, packed, values, wide[:, 2:6], 30, 100, 0.09)
    b.table[:] = -1
    out = check(b, packed, values, wide[:, 2:6], 30, 100, 0.09)
    assert not bool(out.any())


@pytest.mark.parametrize("n,c,back", [([1, 2], [50, 70], 2), ([60], [200], 20), ([5], [60], 3), ([9, 1], [700, 40], 6)])
@pytest.mark.parametrize("hd", [64, 128])
def test_a_group_that_is_not_finite_reaches_the_tokens_that_see_it(dev, n, c, back, hd):
    """A NaN or infinite pair, and codes past f16's range under a finite one (the group's other values count with their weights), in a
    position that the first tokens do not see."""
    b = ref.Batch(n, c, 1, hd, 16, dev, seed=3)
    packed, values = q4(b)
    p = c[0] - back
    words = packed[1].view(torch.int32).view(b.n_pages, -1)
    at = 16 * hd // 8 + 16 + p % 16  # the pair of group 1
    q = torch.randn((b.tokens, 2, hd), generator=torch.Generator().manual_seed(1)).half()
    for d, base in ((float("nan"), 0.0), (float("inf"), 1.0), (1.0, -float("inf")), (900.0, 0.0)):
        pair = torch.tensor([d, base]).half().view(torch.int32)
        words[int(b.table[0, p // 16]), at] = pair.to(dev)
        values[1] = torch.from_numpy(pref.unpack(packed[1].cpu().numpy(), 1)[0]).half()
        _, _, start, ctx, table = b.device()
        got = serving.paged_attention(q.to(dev), *packed, start, ctx, table, max(n), max(c), 0.1).cpu().double()
        want, bound = pref.attention(q, *values, b.start, b.c, b.table, 16, 0.1, 0)
        fine = torch.isfinite(want)
        assert bool((~fine).any()) and bool(torch.equal(fine, torch.isfinite(got)))
        assert bool(((got - want).abs()[fine] <= bound[fine]).all())
        assert torch.equal(want.isnan(), got.isnan()) and torch.equal(want[want.isinf()], got[want.isinf()])


@pytest.mark.parametrize("b,most", [(70, 900), (200, 300), (130, 2500)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 20)])
def test_many_sequences_of_unequal_lengths(dev, b, most, window, sinks):
    """Keys are shared out by what all sequences have: more of them than a wave looks at at once, few long among many short, idle
    ones; with and without the room to cut, and with less of it than the longest would need."""
    rng = np.random.RandomState(b)
    n, c = (rng.rand(b) < 0.9).astype(int), rng.randint(1, 60, b)
    c[rng.randint(0, b, 5)] = most
    n[b // 2:b // 2 + 3] = 2
    batch = ref.Batch(list(n), [int(max(x, y)) for x, y in zip(c, n)], 2, 64, 16, dev, seed=b, extra_tokens=1)
    packed, values = q4(batch)
    q = torch.randn((batch.tokens, 4, 64), generator=torch.Generator().manual_seed(b)).half()
    for max_context, workspace in ((most, None), (64, None), (most, torch.empty(0, dtype=torch.uint8, device=dev)), (10 * most, None)):
        check(batch, packed, values, q, 2, max_context, 0.2, window, sinks, workspace=workspace)


@pytest.mark.parametrize("n,c", [([5, 3], [3, 0]), ([40, 1], [7, 1]), ([2, 1, 60], [1, 0, 200])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (2, 1)])
def test_tokens_before_the_first_position(dev, n, c, window, sinks):
    """More new tokens than positions: those before position 0 see nothing and get zeros, and write nothing."""
    b = ref.Batch(n, c, 2, 64, 16, dev, seed=1)
    packed, values = q4(b)
    q = torch.randn((b.tokens, 4, 64), generator=torch.Generator().manual_seed(1)).half()
    for max_context in (200, 3000):
        out = check(b, packed, values, q, max(n), max_context, 0.1, window, sinks)
        for s in range(len(n)):
            first = int(b.start[s])
            assert not bool(out[first:first + max(0, n[s] - c[s])].any())
    _, _, start, ctx, table = b.device()
    before = [t.clone() for t in packed]
    cos, sin = tables(dev, 256, 64)
    out = torch.full((b.tokens, 4, 64), 9.0, dtype=torch.float16, device=dev)
    serving.qk_rope_append_paged(torch.randn((b.tokens, 8 * 64), device=dev), cos, sin, *packed, start, ctx, table, 4, out=out)
    for s in range(len(n)):
        first, none = int(b.start[s]), max(0, n[s] - c[s])
        assert bool((out[first:first + none] == 9.0).all()) and not bool((out[first + none:int(b.start[s + 1])] == 9.0).all(-1).any())
    if sum(c) == 3:  # a sequence of three positions, all new
        changed = [bool((x != y).view(x.shape[0], -1).any(1)[p]) for x, y in zip(packed, before) for p in range(x.shape[0])]
        assert changed.count(True) <= 2


@pytest.mark.parametrize("max_context", [60, 5000])
def test_starts_that_select_nothing_write_nothing(dev, path, max_context):
    """Starts that fall, lie outside the batch or are all alike: rows of `out` that no sequence has stay as they were."""
    c = [30, 400, 2000]
    b = ref.Batch([4, 3, 2], c, 2, 64, 16, dev, extra_tokens=2)
    packed, _ = q4(b)
    q = torch.randn((b.tokens, 2, 64), generator=torch.Generator().manual_seed(4)).half().to(dev)
    _, _, _, ctx, table = b.device()
    for starts, rows in (([9, 4, 2, 0], []), ([5, 3, -9, -9], []), ([100, 200, 300, 400], []), ([-8, -8, -8, 0], []),
                         ([11, 11, 11, 2 ** 31 - 1], []), ([6, 2, 2, 5], [2, 3, 4]), ([0, 0, 0, 3], [0, 1, 2]), ([3, 1, 4, 4], [1, 2, 3])):
        start = torch.tensor(starts, dtype=torch.int32, device=dev)
        for max_q in (4, 200):
            out = torch.full((b.tokens, 2, 64), 9.0, dtype=torch.float16, device=dev)
            serving.paged_attention(q, *packed, start, ctx, table, max_q, max_context, 0.1, out=out)
            assert bool((out[[t for t in range(b.tokens) if t not in rows]] == 9.0).all()), starts
            serving.paged_attention(q, *packed, start, ctx, table, max_q, max_context, 0.1, window=70, sinks=3, out=out)
            assert bool((out[[t for t in range(b.tokens) if t not in rows]] == 9.0).all()), starts


def test_a_captured_call_shares_out_the_lengths_of_each_replay(dev):
    """Cut contexts, whose cut the device chooses: one graph, other lengths and idle sequences at each replay, against the eager call."""
    b = ref.Batch([1] * 9, [3000] * 9, 2, 128, 16, dev, seed=3)
    packed, _ = q4(b)
    _, _, start, ctx, table = b.device()
    q = torch.randn((9, 8, 128), generator=torch.Generator().manual_seed(1)).half().to(dev)
    call = lambda: serving.paged_attention(q, *packed, start, ctx, table, 1, 3000, 0.1)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    rng = np.random.RandomState(2)
    for i in range(6):
        ctx.copy_(torch.from_numpy(np.minimum(3000, rng.choice([1, 20, 700, 3000], 9) + i)))
        start.copy_(torch.from_numpy(np.concatenate([[0], np.cumsum(rng.rand(9) < 0.8)]).astype(np.int32)))
        rows = int(start[-1])
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got[:rows], call()[:rows]), i


def test_two_calls_at_once(dev):
    """Two streams with calls that are cut, in flight together: the bits of each alone."""
    bs = [ref.Batch([1] * 5, [c] * 5, 2, 64, 16, dev, seed=c) for c in (1500, 2500)]
    args = []
    for b in bs:
        packed, _ = q4(b)
        _, _, start, ctx, table = b.device()
        q = torch.randn((5, 4, 64), generator=torch.Generator().manual_seed(b.c[0])).half().to(dev)
        args.append((q, *packed, start, ctx, table, 1, b.c[0], 0.1))
    want = [serving.paged_attention(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for a, s, g in zip(args, streams, got):
            with torch.cuda.stream(s):
                g.append(serving.paged_attention(*a))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for g, w in zip(got, want) for x in g)


def test_a_captured_step(dev):
    """Append and attention captured once, replayed over other lengths, pages and rows, each replay against the eager call's bits."""
    cos, sin = tables(dev, 512, 128)
    bs = [ref.Batch(n, c, 2, 128, 16, dev, seed=i, spare=40 - sum(-(-x // 16) for x in c)) for i, (n, c) in
          enumerate((([1, 1, 1], [20, 200, 64]), ([1, 0, 1], [33, 9, 300]), ([1, 1, 0], [64, 65, 1])))]
    k, v = (torch.zeros((40, 2, 16, 80), dtype=torch.uint8, device=dev) for _ in range(2))
    start, ctx, table = (torch.zeros(s, dtype=torch.int32, device=dev) for s in (4, 3, (3, 20)))
    qkv = torch.zeros((3, 8 * 128), device=dev)

    def step():
        q = serving.qk_rope_append_paged(qkv, cos, sin, k, v, start, ctx, table, 4, out=torch.zeros((3, 4, 128), dtype=torch.float16, device=dev))
        return serving.paged_attention(q, k, v, start, ctx, table, 1, 300, 0.1, 64, sinks=5, out=torch.zeros_like(q))

    def fill(i):
        b = bs[i]
        for t, new in zip((k, v), q4(b)[0]):
            t.copy_(new)
        start.copy_(torch.from_numpy(b.start))
        ctx.copy_(torch.tensor(b.c, dtype=torch.int32))
        table.fill_(-1)
        table[:, :b.table.shape[1]] = torch.from_numpy(b.table).to(dev)
        qkv.copy_(torch.randn(qkv.shape, generator=torch.Generator().manual_seed(i)))

    fill(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in (0, 1, 2, 0, 2):
        fill(i)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        fill(i)
        assert torch.equal(got, step()), i


def test_another_stream(dev):
    b = ref.Batch([1, 30], [100, 90], 2, 64, 16, dev, seed=5)
    packed, values = q4(b)
    q = torch.randn((b.tokens, 4, 64), generator=torch.Generator().manual_seed(1)).half()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        check(b, packed, values, q, 30, 100, 0.1)
    torch.cuda.current_stream().wait_stream(stream)


def test_refusals(dev, path):
    b = ref.Batch([1, 1], [30, 20], 2, 64, 16, dev)
    (k, v), _ = q4(b)
    _, _, start, ctx, table = b.device()
    q = torch.zeros((2, 4, 64), dtype=torch.float16, device=dev)
    args = start, ctx, table, 1, 30
    for bad, match in (((k, k.half()), "k pages"), ((k[..., :39], v[..., :39]), "contiguous"), ((k[..., :36].contiguous(), v[..., :36].contiguous()), "5 D / 8"),
                       ((k.to(torch.int8), v.to(torch.int8)), "dtype"), ((torch.zeros((4, 2, 16, 20), dtype=torch.uint8, device=dev),) * 2, "over pages")):
        with pytest.raises(DttsError, match=match):
            serving.paged_attention(q, *bad, *args)
    with pytest.raises(DttsError, match="sinks"):
        serving.paged_attention(q, k, v, *args, window=5, sinks=-1)
    with pytest.raises(DttsError, match="misaligned"):
        off = torch.zeros(k.numel() + 8, dtype=torch.uint8, device=dev)[8:].view(k.shape)
        serving.paged_attention(q, off, v, *args)
    with pytest.raises(DttsError, match="page_stride"):
        odd = torch.zeros(4 * (k[0].numel() + 8), dtype=torch.uint8, device=dev).as_strided((4, *k.shape[1:]), (k[0].numel() + 8, *k.stride()[1:]))
        serving.paged_attention(q, odd, odd, *args)
    with pytest.raises(DttsError, match="share memory"):
        cos, sin = tables(dev, 64, 64)
        serving.qk_rope_append_paged(torch.zeros((2, 8 * 64), device=dev), cos, sin, k, k, start, ctx, table, 4)
    with pytest.raises(DttsError, match="dtype"):
        serving.unpack_pages(k.view(torch.float16), v.view(torch.float16))


@pytest.mark.parametrize("apart", [(1 << 31) + 4096, (1 << 32) - 16])
def test_pages_far_apart(dev, apart):
    """Offsets past 31 and 32 bits: the append, attention of single tokens and of a chunk, with sinks and without, the values read
    back and the copy give what they give over neighbouring pages, bit for bit."""
    n, c, n_kv, hd, page = [1, 3, 40], [30, 17, 45], 2, 64, 16
    b = ref.Batch(n, c, n_kv, hd, page, dev, seed=2, spare=0)
    _, _, start, ctx, table = b.device()
    cos, sin = tables(dev, 128, hd)
    qkv = torch.randn((b.tokens, (4 + 2 * n_kv) * hd), generator=torch.Generator().manual_seed(3)).to(dev)
    room = (b.n_pages - 1) * apart + n_kv * page * 40
    near, _ = q4(b)
    far = [torch.empty(room, dtype=torch.uint8, device=dev).as_strided(t.shape, (apart, *t.stride()[1:])) for t in near]
    for f, t in zip(far, near):
        f.copy_(t)
    out = []
    for pages in (near, far):
        q = serving.qk_rope_append_paged(qkv, cos, sin, *pages, start, ctx, table, 4)
        got = [q, *serving.unpack_pages(*pages)]
        for window, sinks in ((0, 0), (20, 5)):
            got.append(serving.paged_attention(q, *pages, start, ctx, table, max(n), max(c), 0.125, window, sinks=sinks))
        ones = torch.arange(3, dtype=torch.int32, device=dev)
        got.append(serving.paged_attention(q[:2].contiguous(), *pages, ones, ctx[[0, 2]], table[[0, 2]], 1, max(c), 0.125))
        move = torch.tensor([b.n_pages - 1, 1], dtype=torch.int32, device=dev), torch.tensor([0, b.n_pages - 2], dtype=torch.int32, device=dev)
        serving.copy_pages(pages, *move)
        got += [t.clone(memory_format=torch.contiguous_format) for t in pages]
        out.append(got)
    for x, y in zip(*out):
        assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


def test_no_tokens(dev, path):
    b = ref.Batch([1], [20], 1, 64, 16, dev, seed=1)
    packed, _ = q4(b)
    before = [t.clone() for t in packed]
    _, _, start, ctx, table = b.device()
    cos, sin = tables(dev, 32, 64)
    q = serving.qk_rope_append_paged(torch.empty((0, 4 * 64), device=dev), cos, sin, *packed, start, ctx, table, 2)
    assert q.shape == (0, 2, 64) and serving.paged_attention(q, *packed, start, ctx, table, 1, 20).shape == q.shape
    none = [torch.zeros(k, dtype=torch.int32, device=dev) for k in (1, 0)]
    q = torch.full((3, 2, 64), 5.0, dtype=torch.float16, device=dev)
    out = serving.paged_attention(q, *packed, *none, table[:0], 1, 20, out=torch.full_like(q, 7.0))
    assert bool((out == 7.0).all()) and all(torch.equal(x, y) for x, y in zip(before, packed))


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,c", [([1], [300]), ([3], [300]), ([40], [300]), ([1, 50, 2], [200, 300, 100])])
@pytest.mark.parametrize("where", ["keys", "values"])
def test_a_missing_page_stands_for_nothing(dev, bits, hd, n, c, where):
    """Blocks without a page, inside the sinks, before and in the window, while page 0 (of no sequence) holds NaN."""
    b = ref.Batch(n, c, 2, hd, 16, dev, seed=hd, extra_tokens=1)
    k, v = (torch.nan_to_num(t, nan=0.5) for t in (b.k, b.v))
    b.table[b.table == 0] = next(i for i in range(1, b.n_pages) if i not in b.table)
    (k if where == "keys" else v)[0] = float("nan")
    b.k, b.v = k, v
    packed, values = q4(b) if bits == 4 else (list(b.device()[:2]), (k, v))
    q = torch.randn((b.tokens, 4, hd), generator=torch.Generator().manual_seed(hd)).half()
    table = b.table
    for block in (0, 1, 2, 5, table.shape[1] - 2):
        b.table = table.copy()
        b.table[:, block] = -1
        for window, sinks in ((0, 0), (1000, 5), (60, 0), (60, 7), (60, 100), (1000, 64)):
            check(b, packed, values, q, max(n), max(c), 0.15, window, sinks)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,c", [([1], [300]), ([1, 2, 4, 0, 3], [700, 2, 90, 40, 333])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200000, 5), (60, 7)])
@pytest.mark.parametrize("bits", [16, 4])
def test_keys_that_no_cache_holds(dev, hd, n, c, window, sinks, bits):
    """A longest context of a million positions makes a call that is taken to read more than the caches keep (short sequences all the
    same), with room for its chunks and without; unseen and missing pages among them."""
    b = ref.Batch(n, c, 2, hd, 16, dev, seed=len(n) + hd, extra_tokens=1)
    b.table[-1, 1:2] = -1
    packed, values = q4(b) if bits == 4 else (list(b.device()[:2]), (b.k, b.v))
    q = torch.randn((b.tokens, 8, hd), generator=torch.Generator().manual_seed(hd)).half()
    for workspace in (None, torch.empty(0, dtype=torch.uint8, device=dev)):
        check(b, packed, values, q, max(n), 1 << 20, 0.15, window, sinks, workspace=workspace)
