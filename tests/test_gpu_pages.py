"""Fork, claim, trim, compact and copy of a cache's pages against plain loops, entry for entry."""
import numpy as np
import pytest
import torch

from dtts import DttsError, serving

import _pages_ref as ref

pytestmark = pytest.mark.gpu

NAMES = ("fork_pages", "claim_pages", "trim_pages", "compact_pages", "copy_pages")


@pytest.fixture(params=["binding", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        for name in NAMES:
            monkeypatch.setattr(serving._serving, name, lambda *args: None)


def up(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)


def host(*tensors):
    return [t.cpu().numpy() for t in tensors]


def pool(seed, b, m, n_pages, share=0.3, waste=0.2):
    """A consistent table and its counts: rows of any length, with pages that earlier rows hold at the same place among them, and
    holes. Some pages of the pool are used by nobody, some counts are under 0."""
    rng = np.random.RandomState(seed)
    ids = list(rng.permutation(n_pages)[:int(n_pages * (1 - waste))])
    table, refs = np.full((b, m), -1, np.int32), np.zeros(n_pages, np.int32)
    for s in range(b):
        for j in range(rng.randint(0, m + 1)):
            r = s and rng.rand() < share
            e = table[rng.randint(0, s), j] if r else ids.pop() if ids and rng.rand() < 0.9 else -1
            table[s, j] = e
            if e >= 0:
                refs[e] += 1
    refs[(refs == 0) & (rng.rand(n_pages) < 0.1)] = -3
    return table, refs, rng


SIZES = [(1, 1, 1), (1, 3, 5), (3, 4, 20), (17, 9, 200), (64, 33, 3000), (300, 5, 1500), (2100, 2, 5000), (2, 700, 1400)]


@pytest.mark.parametrize("b,m,n_pages", SIZES)
def test_fork(dev, path, b, m, n_pages):
    table, refs, rng = pool(b, b, m, n_pages)
    for n in (b, 2 * b + 1, max(1, b // 2)):
        parent = rng.randint(-2, b + 2, n).astype(np.int32)
        parent[: n // 3] = np.arange(n // 3)  # rows that stay
        want = ref.fork(table, refs, parent)
        r = up(refs, dev)
        got = serving.fork_pages(up(table, dev), r, up(parent, dev))
        assert all(np.array_equal(x, y) for x, y in zip(host(got, r), want))
        if n == b:
            t, r = up(table, dev), up(refs, dev)
            assert serving.fork_pages(t, r, up(parent, dev), out=t) is t
            assert all(np.array_equal(x, y) for x, y in zip(host(t, r), want))
            out = torch.empty_like(t)
            assert serving.fork_pages(up(table, dev), up(refs, dev), up(parent, dev), out=out) is out
            assert np.array_equal(out.cpu().numpy(), want[0])


@pytest.mark.parametrize("b,m,n_pages", SIZES)
@pytest.mark.parametrize("page", [16, 64])
def test_claim(dev, path, b, m, n_pages, page):
    table, refs, rng = pool(b + 1, b, m, n_pages, share=0.5)
    for kind in ("decode", "chunks", "beams", "wild"):
        t0, r0 = table.copy(), refs.copy()
        n = (rng.rand(b) < 0.8).astype(int) if kind != "chunks" else rng.randint(0, 3 * page, b)
        c = rng.randint(0, m * page + 2, b)
        if kind == "beams":  # all rows one sequence's
            t0, r0 = ref.fork(t0, r0, np.zeros(b, np.int32))
            c[:] = rng.randint(1, m * page + 1)
        if kind == "wild":
            t0[rng.rand(b, m) < 0.1] = n_pages + 3
            t0[rng.rand(b, m) < 0.1] = rng.randint(0, n_pages)
            c[:: 3] = -5
        start = np.concatenate([[0], np.cumsum(n)])
        if kind == "wild" and b > 2:
            start[2] = 2 ** 31 - 1
        want = ref.claim(t0, r0, start, c, page)
        t, r = up(t0, dev), up(r0, dev)
        src, dst, lacking = serving.claim_pages(t, r, up(start, dev), up(c, dev), page)
        assert all(np.array_equal(x, y) for x, y in zip(host(t, r, src, dst), want)), kind
        assert int(lacking) == want[4], kind


def written(start, c, m, page):
    """The blocks that each row writes to."""
    n, c = np.maximum(np.diff(start), 0), np.minimum(np.maximum(c, 0), m * page)
    first = np.maximum(c - n, 0) // page
    return np.where((n > 0) & (c > 0), -(-c // page) - first, 0)


@pytest.mark.parametrize("b,m,n_pages,share,free_from,n,c,items,need", [
    (3000, 8, 40000, 0.6, 0, (30, 64), (64, 129), (9000, 24000), 4097),  # words and free ids past what LDS holds, shared pages throughout
    (3000, 8, 24000, 0.9, 0, (60, 64), (64, 129), (9000, 24000), 4097),  # most pages shared by many
    (700, 8, 40000, 0.4, 33000, (1, 40), (20, 129), (1025, 4096), 500),  # the free ids far behind, rounds of counts without any
    (1500, 5, 20000, 0.8, 16000, (0, 2), (1, 81), (300, 1024), 100),  # more rows than threads, fewer blocks
    (5000, 3, 60000, 0.5, 50000, (1, 2), (1, 49), (4097, 5000), 1000),  # a token each
])
def test_claim_of_many_blocks(dev, b, m, n_pages, share, free_from, n, c, items, need):
    """Past the sizes that stay in LDS, in a round of threads and in a round of counts; and with a page too few, and with as many as are
    needed to the last."""
    table, refs, rng = pool(b, b, m, n_pages, share=share, waste=0.0)
    refs[:free_from][refs[:free_from] < 1] = 1  # held by other tables
    tokens, ctx = rng.randint(*n, b), rng.randint(*c, b)
    if n == (0, 2):
        tokens = (rng.rand(b) < 0.4).astype(int)
    start = np.concatenate([[0], np.cumsum(tokens)])
    want = ref.claim(table, refs, start, ctx, 16)
    given = int((want[0] != table).sum())
    assert items[0] <= written(start, ctx, m, 16).sum() <= items[1] and given >= need and want[4] == 0
    free = np.flatnonzero(refs < 1)
    for lacking in (0, 1, given // 2):
        r0 = refs.copy()
        r0[free[given - lacking:]] = 1  # held by others
        again = ref.claim(table, r0, start, ctx, 16)
        assert again[4] == lacking
        t, r = up(table, dev), up(r0, dev)
        src, dst, short = serving.claim_pages(t, r, up(start, dev), up(ctx, dev), 16)
        assert all(np.array_equal(x, y) for x, y in zip(host(t, r, src, dst), again)) and int(short) == lacking


def test_claim_of_too_few_pages_changes_nothing(dev):
    table, refs, _ = pool(3, 40, 6, 160, waste=0.0)
    free = int((refs < 1).sum())
    start, c = np.arange(41) * 40, np.full(40, 96)
    want = ref.claim(table, refs, start, c, 16)
    assert want[4] > 0 and free > 0
    t, r = up(table, dev), up(refs, dev)
    src, dst, lacking = serving.claim_pages(t, r, up(start, dev), up(c, dev), 16)
    assert int(lacking) == want[4] and np.array_equal(t.cpu(), table) and np.array_equal(r.cpu(), refs)
    assert bool((src == -1).all()) and bool((dst == -1).all())


@pytest.mark.parametrize("b,m,n_pages", SIZES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 1), (17, 64), (100, 16), (2 ** 31 - 1, 0), (1, 2 ** 31 - 1)])
def test_trim(dev, path, b, m, n_pages, window, sinks):
    table, refs, rng = pool(b + 2, b, m, n_pages)
    c = rng.randint(-5, 16 * m + 20, b)
    want = ref.trim(table, refs, c, 16, window, sinks)
    t, r = up(table, dev), up(refs, dev)
    serving.trim_pages(t, r, up(c, dev), 16, window, sinks)
    assert all(np.array_equal(x, y) for x, y in zip(host(t, r), want))


@pytest.mark.parametrize("b,m,n_pages", SIZES + [(50, 800, 40007), (3, 5, 100000)])
@pytest.mark.parametrize("waste", [0.0, 0.5, 0.95])
def test_compact(dev, path, b, m, n_pages, waste):
    table, refs, _ = pool(b + 3, b, m, n_pages, waste=waste)
    table[table == 0] = n_pages  # entries outside the pool
    want = ref.compact(table, refs)
    t, r = up(table, dev), up(refs, dev)
    src, dst, used = serving.compact_pages(t, r)
    assert all(np.array_equal(x, y) for x, y in zip(host(t, r, src, dst), want)) and int(used) == want[4]
    src, dst, again = serving.compact_pages(t, r)  # nothing is left to move
    assert bool((src == -1).all()) and bool((dst == -1).all()) and int(again) == want[4] and np.array_equal(t.cpu(), want[0])


def test_compact_of_no_and_of_all_pages(dev):
    for refs in ([0] * 70, [1] * 70, [0] * 69 + [1], [1] + [0] * 69):
        refs = np.array(refs, np.int32)
        table = np.arange(70, dtype=np.int32).reshape(7, 10)
        want = ref.compact(table, refs)
        t, r = up(table, dev), up(refs, dev)
        src, dst, used = serving.compact_pages(t, r)
        assert all(np.array_equal(x, y) for x, y in zip(host(t, r, src, dst), want)) and int(used) == want[4]


def test_results_that_are_kept_hold_little_else(dev, path):
    """The parts of one allocation, and a megabyte of scratch at most."""
    table, refs = up(np.full((400, 1000), -1), dev), up(np.zeros(300000), dev)
    start, c = up(np.arange(401), dev), up(np.ones(400), dev)
    for got in (serving.claim_pages(table, refs, start, c, 16), serving.compact_pages(table, refs)):
        for t in got:
            assert t.untyped_storage().nbytes() <= 4 * sum(x.numel() for x in got) + (1 << 20)
    assert sorted(table[:, 0].tolist()) == list(range(400)) and int(refs.sum()) == 400


def test_tables_without_rows(dev, path):
    t, r, one = up(np.zeros((0, 4)), dev), up([1, 0, 2], dev), up([0], dev)
    assert [x.numel() for x in serving.claim_pages(t, r, one, t.view(-1), 16)] == [0, 0, 1]
    assert int(serving.claim_pages(t, r, one, t.view(-1), 16)[2]) == 0
    serving.trim_pages(t, r, t.view(-1), 16, 4)
    assert serving.fork_pages(t, r, t.view(-1)).shape == (0, 4)
    assert serving.fork_pages(t, r, up([0, -1], dev)).tolist() == [[-1] * 4] * 2
    src, dst, used = serving.compact_pages(t, r)
    assert src.tolist() == [2, -1, -1] and dst.tolist() == [1, -1, -1] and int(used) == 2 and r.tolist() == [1, 2, 0]


@pytest.mark.parametrize("n_pages,n", [(3, 1), (50, 20), (300, 120), (2000, 2000)])
def test_copy(dev, path, n_pages, n):
    """Pools of several types and page sizes at once, packed and apart, pages of 16 bytes to 80 KB; what is no destination keeps its bits."""
    rng = np.random.RandomState(n)
    ids = rng.permutation(n_pages)
    pairs = min(n, n_pages // 2)
    src, dst = np.full(n, -1, np.int32), np.full(n, -1, np.int32)
    at = rng.permutation(n)[:pairs]
    src[at], dst[at] = ids[:pairs], ids[pairs:2 * pairs]
    if pairs > 3:
        src[at[0]], dst[at[1]], src[at[2]] = n_pages, -7, 2 ** 31 - 1
    big = max(16, min(256, 4000000 // n_pages // 640) // 16 * 16)
    pools = [torch.rand((n_pages, 2, 16, 64), device=dev).half(), torch.rand((3 * n_pages, 4), device=dev)[::3],
             torch.randint(0, 256, (n_pages, 1, 16, 40), dtype=torch.uint8, device=dev), torch.rand((n_pages, 4, big, 128), device=dev).half()]
    want = [t.clone() for t in pools]
    gaps = pools[1]._base.clone()
    ok = (src >= 0) & (src < n_pages) & (dst >= 0) & (dst < n_pages)
    for t in want:
        t[torch.from_numpy(dst[ok]).long().to(dev)] = t[torch.from_numpy(src[ok]).long().to(dev)]
    serving.copy_pages(pools, up(src, dev), up(dst, dev))
    assert all(torch.equal(x, y) for x, y in zip(pools, want))
    whole = pools[1]._base
    assert torch.equal(whole[1::3], gaps[1::3]) and torch.equal(whole[2::3], gaps[2::3])
    serving.copy_pages(pools[0], up(src, dev), up(dst, dev))  # one pool, again: the same
    assert torch.equal(pools[0], want[0])
    serving.copy_pages([], up(src, dev), up(dst, dev))
    serving.copy_pages(pools, up([], dev), up([], dev))


def test_copy_in_many_layers(dev):
    pools = [torch.rand((9, 2, 16, 64), device=dev).half() for _ in range(130)]
    want = [t.clone() for t in pools]
    for t in want:
        t[3] = t[7]
    serving.copy_pages(pools, up([-1, 7], dev), up([2, 3], dev))
    assert all(torch.equal(x, y) for x, y in zip(pools, want))


def test_captured(dev):
    """One graph of fork, trim, claim, compact and copy, replayed over other tables, counts, lengths and values."""
    b, m, n_pages = 24, 12, 500
    table, refs, parent, start, ctx = (torch.zeros(s, dtype=torch.int32, device=dev) for s in ((b, m), n_pages, b, b + 1, b))
    k = torch.zeros((n_pages, 1, 16, 64), dtype=torch.float16, device=dev)

    def step():
        serving.fork_pages(table, refs, parent, out=table)
        serving.trim_pages(table, refs, ctx, 16, 100, 4)
        src, dst, lacking = serving.claim_pages(table, refs, start, ctx, 16)
        serving.copy_pages([k], src, dst)
        a, c, used = serving.compact_pages(table, refs)
        serving.copy_pages([k], a, c)
        return src, dst, lacking, a, c, used

    def fill(seed):
        t, r, rng = pool(seed, b, m, n_pages, share=0.6)
        for x, y in ((table, t), (refs, r), (parent, rng.randint(-1, b, b)), (start, np.arange(b + 1)), (ctx, rng.randint(1, 16 * m, b))):
            x.copy_(up(y, dev))
        k.copy_(torch.from_numpy(rng.randn(*k.shape)).half())

    fill(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (1, 2, 3, 1):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (table, refs, k, *outs)]
        fill(seed)
        eager = step()
        assert all(torch.equal(x, y) for x, y in zip(got, (table, refs, k, *eager))), seed


def test_refusals(dev, path):
    t, r, p = up(np.zeros((2, 4)), dev), up(np.zeros(9), dev), up([0, 1], dev)
    s = up([0, 1, 2], dev)
    for call, match in (
            (lambda: serving.fork_pages(t.long(), r, p), "dtype"), (lambda: serving.fork_pages(t[:, ::2], r, p), "contiguous"),
            (lambda: serving.fork_pages(t.cpu(), r, p), "on the device"), (lambda: serving.fork_pages(t[0], r, p), "max_pages"),
            (lambda: serving.fork_pages(t, r, p, out=up(np.zeros((2, 5)), dev)), "is not"),
            (lambda: serving.fork_pages(t, r, p, out=t, workspace=torch.empty(31, dtype=torch.uint8, device=dev)), "workspace"),
            (lambda: serving.fork_pages(t, t.view(-1), p), "share memory"), (lambda: serving.fork_pages(t, r, r), "share memory"),
            (lambda: serving.fork_pages(t, r, p[:1], out=t[1:]), "no part"),
            (lambda: serving.claim_pages(t, r, p, p, 16), "q_start"), (lambda: serving.claim_pages(t, r, s, s, 16), "context"),
            (lambda: serving.claim_pages(t, r, s, p, 24), "power of two"), (lambda: serving.claim_pages(t, r, s, p, 8), "power of two"),
            (lambda: serving.claim_pages(t, r, s, p, 16, workspace=torch.empty(8, dtype=torch.uint8, device=dev)), "workspace"),
            (lambda: serving.claim_pages(t, r[:0], s, p, 16), "pages"),
            (lambda: serving.trim_pages(t, r, p, 16, 0), "window"), (lambda: serving.trim_pages(t, r, p, 16, 5, -1), "sinks"),
            (lambda: serving.trim_pages(t, r, s, 16, 5), "context"),
            (lambda: serving.compact_pages(t, r.view(3, 3)), "n_pages"),
            (lambda: serving.compact_pages(t, r, workspace=torch.empty(8, dtype=torch.uint8, device=dev)), "workspace"),
            (lambda: serving.copy_pages([torch.zeros((4, 3), device=dev)], p, p), "multiples of 16"),
            (lambda: serving.copy_pages([torch.zeros((4, 8), device=dev)[:, ::2]], p, p), "contiguous pages"),
            (lambda: serving.copy_pages([torch.zeros((4, 8), device=dev), torch.zeros((5, 8), device=dev)], p, p), "contiguous pages"),
            (lambda: serving.copy_pages([torch.zeros((1, 8), device=dev).expand(4, 8)], p, p), "multiples of 16"),
            (lambda: serving.copy_pages([torch.zeros((4, 8))], p, p), "on the device"),
            (lambda: serving.copy_pages([torch.zeros((4, 8), device=dev)], p, s), "destinations")):
        with pytest.raises(DttsError, match=match):
            call()
