"""Windows with first tokens that stay visible, over f16 pages, against 64-bit evaluations (tests of 4-bit pages: test_gpu_q4_cache)."""
import pytest
import torch

from dtts import serving

import _pages_ref as pref
import _serving_ref as ref

pytestmark = pytest.mark.gpu


def check(b, q, max_q, max_context, scale, window, sinks, **more):
    k, v, start, ctx, table = b.device()
    q = q.to(b.dev)
    out = torch.full((b.tokens, q.shape[1], b.hd), 9.0, dtype=torch.float16, device=b.dev)
    got = serving.paged_attention(q, k, v, start, ctx, table, max_q, max_context, scale, window, out=out, sinks=sinks, **more)
    t = int(b.start[-1])
    want, bound = pref.attention(q, b.k, b.v, b.start, b.c, b.table, b.page, scale, window, sinks)
    fine = torch.isfinite(want[:t])
    err = (got[:t].cpu().double() - want[:t]).abs()
    assert bool(torch.equal(fine, torch.isfinite(got[:t].cpu())))
    assert bool((err[fine] <= bound[:t][fine]).all()), f"{(err[fine] / bound[:t][fine]).max()} of the bound"
    assert bool((got[t:] == 9.0).all())
    return got


SEQS = [([1], [1]), ([1, 1, 0, 1], [700, 63, 20, 65]), ([2, 9], [300, 9]), ([50, 1], [400, 800]), ([130], [130]), ([70], [1000])]


@pytest.mark.parametrize("n,c", SEQS)
@pytest.mark.parametrize("window,sinks", [(1, 1), (2, 64), (31, 4), (64, 63), (65, 128), (128, 1), (200, 130), (7, 5000)])
def test_sinks(dev, n, c, window, sinks):
    """Sinks within a key tile and past several, windows that reach them and windows far behind."""
    hd = 128 if window % 2 else 64
    b = ref.Batch(n, c, 2, hd, 16 if sinks % 2 else 64, dev, seed=sinks, extra_tokens=1)
    q = torch.randn((b.tokens, 6, hd), generator=torch.Generator().manual_seed(window)).half()
    for max_q in (max(n), 1):
        check(b, q, max_q, max(c), 0.3, window, sinks)


@pytest.mark.parametrize("n", [1, 40])
def test_many_chunks(dev, n):
    """A cut axis: chunks that hold the sinks' end, the gap and windows, joined."""
    b = ref.Batch([n], [5000], 1, 64, 32, dev, seed=n)
    q = torch.randn((n, 2, 64), generator=torch.Generator().manual_seed(n)).half()
    for window, sinks in ((2000, 1000), (900, 4), (3000, 2500), (1500, 700)):
        check(b, q, n, 5000, 0.1, window, sinks)
        check(b, q, n, 5000, 0.1, window, sinks, workspace=torch.empty(0, dtype=torch.uint8, device=dev))


def test_pages_between_sinks_and_window_are_free(dev):
    """The pages that trim_pages frees are no page of any key that is seen: the same bits without them."""
    b = ref.Batch([1, 1, 20], [800, 90, 600], 2, 128, 16, dev, seed=2)
    k, v, start, ctx, table = b.device()
    q = torch.randn((b.tokens, 4, 128), generator=torch.Generator().manual_seed(1)).half().to(dev)
    want = serving.paged_attention(q, k, v, start, ctx, table, 20, 800, 0.1, 64, sinks=5)
    refs = torch.zeros(b.n_pages, dtype=torch.int32, device=dev)
    refs[table[table >= 0].long()] = 1
    trimmed = table.clone()
    serving.trim_pages(trimmed, refs, ctx - torch.tensor([1, 1, 20], dtype=torch.int32, device=dev), 16, 64, sinks=5)
    assert int((refs == 0).sum()) > 60 and int((trimmed == -1).sum()) > int((table == -1).sum())
    gone = refs == 0
    k[gone], v[gone] = float("nan"), float("nan")
    assert torch.equal(serving.paged_attention(q, k, v, start, ctx, trimmed, 20, 800, 0.1, 64, sinks=5), want)


@pytest.mark.parametrize("n,c", [([1], [400]), ([1, 3], [200, 300]), ([60], [400])])
def test_values_that_are_not_finite(dev, n, c):
    """NaN among the sinks, between them and the window, and in the window: each in the tokens that see it alone."""
    for p, window, sinks in ((2, 50, 4), (5, 50, 4), (70, 50, 66), (c[0] - 3, 50, 4), (c[0] - 55, 50, 1), (c[0] - 80, 50, 70)):
        b = ref.Batch(n, c, 1, 64, 16, dev, seed=4)
        b.v[b.table[0, p // 16], :, p % 16, 3::7] = float("nan")
        b.v[b.table[0, p // 16], :, p % 16, 4::7] = float("inf")
        q = torch.randn((b.tokens, 2, 64), generator=torch.Generator().manual_seed(1)).half()
        check(b, q, max(n), max(c), 0.1, window, sinks)


def test_sinks_without_a_window_count_for_nothing(dev):
    b = ref.Batch([1, 40], [100, 90], 1, 64, 16, dev, seed=1)
    k, v, start, ctx, table = b.device()
    q = torch.randn((b.tokens, 2, 64), generator=torch.Generator().manual_seed(1)).half().to(dev)
    want = serving.paged_attention(q, k, v, start, ctx, table, 40, 100, 0.1)
    for window, sinks in ((0, 7), (2 ** 30, 7), (0, 2 ** 31 - 1), (100, 2 ** 31 - 1), (1, 2 ** 30)):
        got = serving.paged_attention(q, k, v, start, ctx, table, 40, 100, 0.1, window, sinks=sinks)
        assert torch.equal(got, want) or (window in (1, 100) and bool(((got - want).abs().double() <= 2.0 ** -10 * want.abs() + 2.0 ** -10).all()))
