"""dtts_qk_rope_append_paged_* and dtts_paged_attention_f16 against 64-bit references over ragged batches:
pools whose unused slots are NaN, idle slots, chunks and single tokens, windows, pages that end inside a
tile, contexts shorter than their chunk, missing pages, values that are not finite."""
import numpy as np
import pytest
import torch

from dtts import DttsError, ops, serving

import _serving_ref as ref

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- append

def _append_case(dev, b, heads, dtype, norm, rot, seed=0, length=700):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn((b.tokens, (heads + 2 * b.n_kv) * b.hd), generator=g).to(dtype).to(dev)
    norms = (torch.rand((2, b.hd), generator=g) * 0.4 + 0.8).to(dev) if norm else None
    cos, sin = (torch.from_numpy(t).to(dev) for t in ops.rope_table_f32(length, rot, 1e4))
    return qkv, norms, cos, sin


def _append_want(b, heads, qkv, norms, cos, sin, interleaved, eps):
    """Per token of a sequence: (row, sequence, position, turned q|k and v, their bounds) in 64 bits."""
    x = qkv.cpu().double().numpy().reshape(b.tokens, heads + 2 * b.n_kv, b.hd)
    seq = np.repeat(np.arange(len(b.n)), b.n)
    i = np.concatenate([np.arange(n) for n in b.n]) if len(seq) else np.zeros(0, int)
    pos = np.array(b.c)[seq] - np.array(b.n)[seq] + i
    qk = x[:len(seq), :heads + b.n_kv].copy()
    if norms is not None:
        w = norms.cpu().double().numpy()
        qk[:, :heads] = ref.rms(qk[:, :heads], w[0], eps)
        qk[:, heads:] = ref.rms(qk[:, heads:], w[1], eps)
    ok = (pos >= 0) & (pos < cos.shape[0])
    at = np.clip(pos, 0, cos.shape[0] - 1)
    y, mag = ref.turn(qk, cos.cpu().double().numpy()[at], sin.cpu().double().numpy()[at], interleaved)
    # f32: the norm's sum of 128 squares (8 in order, then 4 levels), root, two products and the division (20
    # roundings in all), the turn's three; then f16
    tol = 24 * 2.0 ** -24 * mag + 2.0 ** -11 * np.abs(y) * (1 + 2.0 ** -10) + 2.0 ** -25
    return seq, pos, ok, y, tol, x[:len(seq), heads + b.n_kv:]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("n,c,heads,n_kv,hd,rot,page,interleaved,norm", [
    ([1], [1], 1, 1, 64, 64, 16, False, False),
    ([1] * 48, list(range(1, 480, 10)), 16, 8, 128, 128, 16, False, True),
    ([5, 0, 130, 1, 0, 33], [5, 7, 300, 64, 0, 40], 4, 2, 128, 64, 32, False, True),
    ([17, 1, 100], [17, 65, 200], 10, 2, 64, 16, 64, True, True),
    ([3, 2], [131, 2], 5, 1, 64, 64, 128, True, False),
    ([0, 0, 0, 9], [0, 16, 3, 600], 2, 2, 128, 8, 16, False, False),
])
def test_append(dev, n, c, heads, n_kv, hd, rot, page, interleaved, norm, dtype):
    b = ref.Batch(n, c, n_kv, hd, page, dev, seed=len(n), extra_tokens=3)
    qkv, norms, cos, sin = _append_case(dev, b, heads, dtype, norm, rot)
    k, v, start, ctx, table = b.device()
    kw, vw = k.cpu().double().numpy(), v.cpu().double().numpy()
    out = torch.full((b.tokens, heads, hd), 9.0, dtype=torch.float16, device=dev)
    got = serving.qk_rope_append_paged(qkv, cos, sin, k, v, start, ctx, table, heads, norms, 1e-5, interleaved, out)
    seq, pos, ok, y, tol, vv = _append_want(b, heads, qkv, norms, cos, sin, interleaved, 1e-5)
    q = got.cpu().double().numpy()
    assert np.all(np.abs(q[:len(seq)] - y[:, :heads]) <= tol[:, :heads])
    assert np.all(q[len(seq):] == 9.0), "rows of no sequence were written"
    kt = np.zeros_like(kw)
    for t, (s, p) in enumerate(zip(seq, pos)):
        at = b.table[s, p // page], slice(None), p % page
        kw[at], kt[at], vw[at] = y[t, heads:], tol[t, heads:], vv[t].astype(np.float32).astype(np.float16)
    kg, vg = k.cpu().double().numpy(), v.cpu().double().numpy()
    assert np.array_equal(np.isnan(kg), np.isnan(kw)) and np.all((np.abs(kg - kw) <= kt) | np.isnan(kw))
    assert np.array_equal(vg, vw, equal_nan=True)


def test_append_matches_the_rectangular_form(dev):
    """One token a lane, half split, whole head: the queries and the cache rows of
    dtts_qk_norm_rope_kv_append_f32, rounded, within one f16 step (its norm divides where this multiplies)."""
    lanes, heads, n_kv, hd, page, cap = 7, 8, 4, 128, 16, 64
    c = [1, 17, 16, 33, 64, 5, 40]
    b = ref.Batch([1] * lanes, c, n_kv, hd, page, dev)
    qkv, norms, cos, sin = _append_case(dev, b, heads, torch.float32, True, hd)
    k, v, start, ctx, table = b.device()
    q = serving.qk_rope_append_paged(qkv, cos, sin, k, v, start, ctx, table, heads, norms, 1e-6)
    rk, rv = (torch.zeros((lanes, n_kv, cap, hd), dtype=torch.float16, device=dev) for _ in range(2))
    want = ops.qk_norm_rope_kv_append(qkv, norms, cos, sin, np.array(c) - 1, rk, rv, heads, 1e-6).half()

    def near(x, y):
        return bool(((x.float() - y.float()).abs() <= 2.0 ** -10 * y.float().abs() + 2.0 ** -24).all())

    assert near(q, want)
    for s in range(lanes):
        at = b.table[s, (c[s] - 1) // page], slice(None), (c[s] - 1) % page
        assert near(k[at], rk[s, :, c[s] - 1]) and torch.equal(v[at], rv[s, :, c[s] - 1])


def test_append_leaves_out_tokens_without_a_place(dev):
    """Positions below 0 (a context shorter than its chunk) and past the table, missing and impossible pages,
    impossible starts: nothing of such a token is written."""
    n, c = [4, 3, 2, 2, 2], [2, 30, 40, 20, 9]
    b = ref.Batch(n, c, 2, 64, 16, dev, extra_tokens=2)
    b.table[1, 1], b.table[2, 2], b.table[3, 1] = -7, b.n_pages, 2 ** 31 - 1
    heads = 2
    qkv, norms, cos, sin = _append_case(dev, b, heads, torch.float32, True, 64, length=9)
    cos30, sin30 = (torch.from_numpy(t).to(dev) for t in ops.rope_table_f32(64, 64, 1e4))
    for tab in ((cos30, sin30), (cos, sin)):
        k, v, start, ctx, table = b.device()
        before = k.clone(), v.clone()
        out = torch.full((b.tokens, heads, 64), 9.0, dtype=torch.float16, device=dev)
        serving.qk_rope_append_paged(qkv, *tab, k, v, start, ctx, table, heads, norms, 1e-6, out=out)
        skipped = (out == 9.0).flatten(1).all(1).cpu().tolist()
        # sequence 0: positions -2, -1, 0, 1; 1: 27..29 on a missing page; 2: 38, 39 on one; 3: 18, 19; 4: 7, 8
        assert skipped == [True, True, False, False] + [True] * 7 + [False, False] + [True] * 2
        changed = (k != before[0]) & ~(torch.isnan(k) & torch.isnan(before[0]))
        assert int(changed.flatten(2).any(2).any(1).sum()) == 2  # sequence 0's page and 4's
    # starts that fall, and pass the batch: no access outside it, and untouched where nothing is selected
    k, v, start, ctx, table = b.device()
    start[:] = torch.tensor([5, 3, -9, 100, 2 ** 31 - 1, 7], dtype=torch.int32)
    out = torch.full((b.tokens, heads, 64), 9.0, dtype=torch.float16, device=dev)
    serving.qk_rope_append_paged(qkv, cos30, sin30, k, v, start, ctx, table, heads, norms, 1e-6, out=out)
    torch.cuda.synchronize()


# ---------------------------------------------------------------- attention

def _queries(b, heads, dev, seed=1, scale=1.3):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((b.tokens, heads, b.hd), generator=g) * scale).half().to(dev)


def _attend(b, q, dev, scale, window=0, max_q=None, max_context=None, split=True, dirty=True, arrays=None):
    k, v, start, ctx, table = arrays or b.device()
    out = torch.full(q.shape, 9.0, dtype=torch.float16, device=dev)
    max_q, max_context = max_q or max(max(b.n), 1), max_context or max(max(b.c), 1)
    need = serving.paged_attention_workspace_bytes(b.tokens, len(b.n), q.shape[1], b.n_kv, b.hd, max_q, max_context, window)
    # a workspace of NaN: what is not written is not read
    ws = torch.full((max(need, 16) // 4,), float("nan"), device=dev).view(torch.uint8) if split else torch.empty(0, dtype=torch.uint8, device=dev)
    serving.paged_attention(q, k, v, start, ctx, table, max_q, max_context, scale, window, out, ws)
    want, tol = ref.attention(q, k, v, b.start, b.c, b.table, b.page, scale, window)
    used = int(b.start[-1])
    got = out.cpu().double()
    assert bool((got[used:] == 9.0).all()), "rows of no sequence were written"
    bad = ~((got[:used] - want[:used]).abs() <= tol[:used]) & ~(got[:used].isnan() & want[:used].isnan())
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:3].tolist(), float((got[:used] - want[:used]).abs().nan_to_num(0).max()))
    return out


CASES = [
    # one token over contexts around tile and page ends
    ([1] * 8, [1, 2, 15, 16, 17, 31, 33, 65], 16, 8, 128, 16, 0),
    ([1] * 6, [63, 64, 65, 127, 128, 129], 2, 2, 64, 64, 0),
    # uneven head groups, an idle slot, an empty sequence
    ([1, 0, 1, 0, 1], [300, 17, 41, 0, 700], 10, 2, 128, 32, 0),
    ([1, 1], [2000, 900], 8, 1, 64, 16, 0),
    # chunks: prompts from nothing, after a prefix, beside single tokens
    ([37], [37], 4, 2, 128, 16, 0),
    ([100, 1, 3, 0, 17], [100, 333, 40, 12, 500], 8, 2, 64, 32, 0),
    ([130, 129, 1], [130, 400, 129], 4, 4, 128, 128, 0),
    ([64, 65], [64, 65], 5, 1, 128, 16, 0),
    # windows: shorter than a tile, inside one, longer than the context
    ([1] * 4, [5, 80, 300, 1000], 4, 2, 128, 16, 7),
    ([50, 1, 200], [300, 300, 200], 4, 2, 64, 16, 33),
    ([150, 1], [700, 90], 2, 1, 128, 64, 1),
    ([70], [500], 2, 2, 64, 32, 4000),
]


@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("n,c,heads,n_kv,hd,page,window", CASES)
def test_attention(dev, n, c, heads, n_kv, hd, page, window, split):
    b = ref.Batch(n, c, n_kv, hd, page, dev, seed=len(c), extra_tokens=2)
    _attend(b, _queries(b, heads, dev), dev, hd ** -0.5, window, split=split)


@pytest.mark.parametrize("max_q,max_context", [(1, 1), (1, 64), (4000, 60000), (7, 300)])
def test_attention_whatever_the_caller_says_of_lengths(dev, max_q, max_context):
    """max_q and max_context size the launch only: contexts and chunks past them, or far under, come out the
    same within the same bound."""
    b = ref.Batch([40, 1, 0, 9], [1500, 700, 9, 9], 2, 128, 16, dev)
    _attend(b, _queries(b, 4, dev), dev, 0.1, max_q=max_q, max_context=max_context)


def test_attention_many_sequences(dev):
    """More sequences than a wave has lanes, some of them idle, single tokens and short chunks."""
    rng = np.random.RandomState(3)
    n = [int(x) for x in rng.choice([0, 1, 1, 1, 2, 9, 40], 150)]
    c = [x + int(rng.randint(0, 90)) for x in n]
    b = ref.Batch(n, c, 1, 64, 16, dev)
    _attend(b, _queries(b, 3, dev), dev, 0.125)


def test_attention_contexts_shorter_than_their_chunk_and_empty_ones(dev):
    """Tokens before position 0 see nothing: zeros."""
    n, c = [5, 3, 2, 140], [2, 0, 30, 20]
    b = ref.Batch(n, c, 2, 64, 16, dev)
    out = _attend(b, _queries(b, 4, dev), dev, 0.125)
    assert bool((out[:3] == 0).all()) and bool((out[5:8] == 0).all()) and bool((out[10:130] == 0).all())
    b.c = [-5, -2 ** 31, 30, 20]
    _attend(b, _queries(b, 4, dev), dev, 0.125, max_context=30)


@pytest.mark.parametrize("n", [[1, 1, 1], [60, 1, 200]])
def test_attention_without_a_page(dev, n):
    """Positions whose page id is missing or impossible are not attended to; a row with none left is zero.
    A context past the page table ends with it."""
    c = [200, 30, 250]
    b = ref.Batch(n, c, 2, 64, 16, dev)
    b.table[0, 3], b.table[0, 7], b.table[2, 0] = -1, b.n_pages, -2 ** 31
    b.table[1, :] = -1
    out = _attend(b, _queries(b, 4, dev), dev, 0.125)
    assert bool((out[n[0]] == 0).all())
    b = ref.Batch(n, c, 2, 64, 16, dev)
    b.c[2] = 20000  # the table's width is 16 pages
    if n[2] == 1:
        _attend(b, _queries(b, 4, dev), dev, 0.125)


@pytest.mark.parametrize("n,c", [([1, 1], [40, 300]), ([90, 1], [100, 300]), ([200], [200])])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_attention_a_value_that_is_not_finite_reaches_only_who_sees_it(dev, n, c, value):
    b = ref.Batch(n, c, 2, 128, 16, dev)
    hit = c[0] - n[0] // 2 - 1  # the middle token of the first sequence's chunk (or its only one)
    arrays = b.device()
    for t, head in ((arrays[1], 0), (arrays[0], 1)):
        t[b.table[0, hit // 16], head, hit % 16, 5] = value
    q = _queries(b, 4, dev)
    out = torch.empty_like(q)
    serving.paged_attention(q, *arrays, max(n), max(c), 0.1, out=out)
    clean = torch.empty_like(q)
    k, v, *rest = b.device()
    serving.paged_attention(q, k, v, *rest, max(n), max(c), 0.1, out=clean)
    first = n[0] - n[0] // 2 - 1 if n[0] > 1 else 0  # the first row that sees it
    assert bool(torch.isfinite(out[:first]).all()) and bool(torch.isfinite(out[n[0]:]).all())
    assert bool((out[:first].float() - clean[:first].float()).abs().le(2.0 ** -9 * clean[:first].float().abs() + 2.0 ** -9).all())
    assert torch.equal(out[n[0]:], clean[n[0]:])
    seen = out[first:n[0], 0:2, 5]  # value heads' dimension 5: not finite wherever the weight is not 0
    assert not bool(torch.isfinite(seen).any())


def test_attention_large_scores(dev):
    """Scores in the thousands, one key far ahead of the rest, and all equal."""
    b = ref.Batch([1, 40], [500, 300], 2, 128, 16, dev)
    q = _queries(b, 4, dev, scale=30.0)
    out = _attend(b, q, dev, 1.0)
    assert bool(torch.isfinite(out).all())
    k, v, start, ctx, table = b.device()
    k.nan_to_num_(0).zero_()
    got = serving.paged_attention(q, k, v, start, ctx, table, 40, 500, 1.0)
    want, tol = ref.attention(q, k, v, b.start, b.c, b.table, 16, 1.0, 0)
    assert bool(((got.cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("scale", [-0.1, 0.0, -3.0, 1e-30])
def test_attention_scales(dev, scale):
    """A negative scale, none at all, one that leaves every weight equal."""
    b = ref.Batch([1, 60, 2], [100, 200, 700], 2, 64, 16, dev)
    _attend(b, _queries(b, 4, dev), dev, scale)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 30, 2 ** 30 - 1])
def test_attention_windows_past_every_position(dev, window):
    """With contexts shorter than their chunks, whose first tokens are before position 0."""
    b = ref.Batch([200, 3, 60], [100, 3, 300], 2, 64, 16, dev)
    _attend(b, _queries(b, 4, dev), dev, 0.1, window)


@pytest.mark.parametrize("window", [0, 1, 7])
@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 30 + 2 ** 24 + 1, 2 ** 30 + 40, 2 ** 30, -1, -2 ** 31 + 1, -2 ** 31])
def test_attention_of_impossible_lengths(dev, length, window):
    """Positions no table holds, at the ends of an int: the chunk and the single token of such a length end, and
    their neighbours are right. (A window's first key, rounded and 96 further, passed the int's end: the waves
    then walked 2^31 keys.)"""
    b = ref.Batch([1, 1, 50, 20], [60, 70, 100, 30], 2, 64, 16, dev)
    b.c[1] = b.c[2] = length
    _attend(b, _queries(b, 4, dev), dev, 0.1, window)


@pytest.mark.parametrize("n", [[8, 1, 8], [9, 8, 1], [8, 7, 9, 17]])
def test_attention_at_the_rows_that_choose_the_tile(dev, n):
    """Four query heads a kv head: 32 rows of a sequence are the small tiles' last, 36 the large ones' first."""
    b = ref.Batch(n, [x + 70 for x in n], 2, 128, 16, dev)
    _attend(b, _queries(b, 8, dev), dev, 0.1)


@pytest.mark.parametrize("c", [[900, 50, 0, 385], [2000, 129, 1500, 1]])
@pytest.mark.parametrize("heads", [3, 6])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_joins_chunks_of_odd_and_even_heads(dev, c, heads, hd):
    """Up to eight chunks a row and more, rows with one or none beside them, padding behind."""
    b = ref.Batch([1, 1, 0, 2], c, 3, hd, 16, dev, extra_tokens=2)
    _attend(b, _queries(b, heads, dev), dev, 0.1)


def test_sequences_share_a_prefix(dev):
    """Three sequences over the pages of one prefix and their own last page."""
    b = ref.Batch([1, 20, 1], [70, 84, 66], 2, 128, 16, dev)
    for s in (1, 2):
        b.table[s, :4] = b.table[0, :4]
    _attend(b, _queries(b, 4, dev), dev, 0.1)


def test_attention_starts_that_do_not_rise(dev):
    """Nonsense in q_start selects nothing outside the batch: the call ends, and later calls are right."""
    b = ref.Batch([9, 1, 40], [90, 10, 100], 2, 64, 16, dev)
    k, v, start, ctx, table = b.device()
    q = _queries(b, 4, dev)
    want = serving.paged_attention(q, k, v, start, ctx, table, 40, 100, 0.1)
    for bad in ([50, 0, 50, 0], [-5, 99, -5, 99], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 0], [0, 50, 50, 50]):
        odd = torch.tensor(bad, dtype=torch.int32, device=dev)
        serving.paged_attention(q, k, v, odd, ctx, table, 40, 100, 0.1)
        serving.paged_attention(q, k, v, odd, ctx, table, 1, 2000, 0.1)
    assert torch.equal(serving.paged_attention(q, k, v, start, ctx, table, 40, 100, 0.1), want)


def test_attention_strided_queries_and_pages(dev):
    """Queries inside a qkv tensor; pages of every third place of a larger pool."""
    b = ref.Batch([3, 1, 70], [90, 300, 100], 2, 64, 32, dev, stride_pages=3)
    wide = torch.randn((b.tokens, 8 + 4, 64), generator=torch.Generator().manual_seed(2)).half().to(dev)
    arrays = b.device()
    got = serving.paged_attention(wide[:, :8], *arrays, 70, 300, 0.125)
    want, tol = ref.attention(wide[:, :8], arrays[0], arrays[1], b.start, b.c, b.table, 32, 0.125, 0)
    assert bool(((got.cpu().double() - want).abs() <= tol).all())
    assert torch.equal(got, serving.paged_attention(wide[:, :8].contiguous(), *arrays, 70, 300, 0.125))


def test_append_and_attention_past_4_gib(dev):
    """A pool whose last pages lie past 2^32 bytes, and past 2^31 elements."""
    n_pages, n_kv, page, hd, heads = 17001, 8, 128, 128, 8  # 4.46 GB a tensor, 2.2e9 elements
    k, v = (torch.zeros((n_pages, n_kv, page, hd), dtype=torch.float16, device=dev) for _ in range(2))
    b = ref.Batch([1, 130], [200, 300], n_kv, hd, page, dev)
    sk, sv, start, ctx, table = b.device()
    moved = torch.where(table >= 0, n_pages - 1 - table, table).contiguous()
    for s in range(2):
        for p in table[s].tolist():
            if p >= 0:
                k[n_pages - 1 - p], v[n_pages - 1 - p] = sk[p], sv[p]
    qkv, norms, cos, sin = _append_case(dev, b, heads, torch.float16, True, hd)
    q1 = serving.qk_rope_append_paged(qkv, cos, sin, sk, sv, start, ctx, table, heads, norms)
    q2 = serving.qk_rope_append_paged(qkv, cos, sin, k, v, start, ctx, moved, heads, norms)
    assert torch.equal(q1, q2)
    o1 = serving.paged_attention(q1, sk, sv, start, ctx, table, 130, 300, 0.1)
    o2 = serving.paged_attention(q2, k, v, start, ctx, moved, 130, 300, 0.1)
    assert torch.equal(o1, o2) and bool(torch.isfinite(o1).all())


def test_sizes_given_as_numpy_numbers(dev):
    b = ref.Batch([3, 40], [90, 300], 2, 64, 16, dev)
    k, v, start, ctx, table = b.device()
    q = _queries(b, 4, dev)
    want = serving.paged_attention(q, k, v, start, ctx, table, 40, 300, 0.125, 100)
    got = serving.paged_attention(q, k, v, start, ctx, table, np.int64(40), np.int32(300), np.float32(0.125), np.int64(100))
    assert torch.equal(got, want)


def test_paged_python_refusals(dev):
    b = ref.Batch([1, 2], [20, 30], 2, 64, 16, dev)
    k, v, start, ctx, table = b.device()
    q = _queries(b, 4, dev)
    with pytest.raises(DttsError, match="over pages of head_dim"):
        serving.paged_attention(q[..., :32].contiguous(), k, v, start, ctx, table, 2, 30)
    with pytest.raises(DttsError, match="contiguous rows"):
        serving.paged_attention(q[..., ::2], k, v, start, ctx, table, 2, 30)
    with pytest.raises(DttsError, match="heads over"):
        serving.paged_attention(q[:, :3].contiguous(), k, v, start, ctx, table, 2, 30)
    with pytest.raises(DttsError, match="dtype"):
        serving.paged_attention(q, k, v, start.long(), ctx, table, 2, 30)
    with pytest.raises(DttsError, match="pages"):
        serving.paged_attention(q, k, v[:-1], start, ctx, table, 2, 30)
    with pytest.raises(DttsError, match="page table"):
        serving.paged_attention(q, k, v, start[:-1], ctx, table, 2, 30)
    with pytest.raises(DttsError, match="a page must be contiguous"):
        serving.paged_attention(q, k.transpose(1, 2), v.transpose(1, 2), start, ctx, table, 2, 30)
    with pytest.raises(DttsError, match="qkv"):
        serving.qk_rope_append_paged(q.view(3, -1), torch.zeros((9, 32), device=dev), torch.zeros((9, 32), device=dev), k, v, start,
                                     ctx, table, 4)
