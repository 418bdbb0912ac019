"""Calls of dtts.serving that the documentation allows and a tensor's form makes unusual; through the binding and through
Python alone."""
import pytest
import torch

from dtts import DttsError, serving

import _serving_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["binding", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        for name in ("rotary", "qk_rope_append_paged", "paged_attention", "sample"):
            monkeypatch.setattr(serving._serving, name, lambda *args: None)


def _odd_strides(t, dim):
    """t with another number as the stride of its size of 1 at `dim`, as transposes and slices leave it."""
    stride = list(t.stride())
    stride[dim] = 24
    y = t.as_strided(t.shape, stride)
    assert y.is_contiguous() and y.stride() != t.stride()
    return y


def test_the_stride_of_a_size_of_one_is_no_ones(dev, path):
    """One head, one kv head, one row, one page: contiguous tensors, whatever torch has as that stride."""
    g = torch.Generator().manual_seed(2)
    b = ref.Batch([3, 1], [40, 90], 1, 64, 16, dev)
    k, v, *rest = b.device()
    q = torch.randn((b.tokens, 1, 64), generator=g).half().to(dev)
    want = serving.paged_attention(q, k, v, *rest, 3, 90, 0.1)
    assert torch.equal(serving.paged_attention(_odd_strides(q, 1), _odd_strides(k, 1), _odd_strides(v, 1), *rest, 3, 90, 0.1), want)
    assert torch.equal(serving.paged_attention(q, _odd_strides(k, 1), v, *rest, 3, 90, 0.1), want)  # k's and v's need not agree
    one = ref.Batch([1], [10], 2, 64, 16, dev, spare=0)
    k, v, *rest = one.device()
    q = torch.randn((1, 4, 64), generator=g).half().to(dev)
    want = serving.paged_attention(q, k, v, *rest, 1, 10, 0.1)
    assert k.shape[0] == 1 and torch.equal(serving.paged_attention(_odd_strides(q, 0), _odd_strides(k, 0), v, *rest, 1, 10, 0.1), want)

    cos, sin = (torch.from_numpy(t).to(dev) for t in serving.rope_table_scaled(128, 64, 1e4))
    for shape, dim in (((5, 1, 64), 1), ((1, 4, 64), 0)):
        x, pos = torch.randn(shape, generator=g).to(dev), torch.arange(shape[0], dtype=torch.int32, device=dev) + 7
        want = serving.rotary(x, cos, sin, pos)
        assert torch.equal(serving.rotary(_odd_strides(x, dim), cos, sin, pos), want)
        out = _odd_strides(torch.zeros_like(x), dim)
        assert torch.equal(serving.rotary(x, cos, sin, pos, out=out), want)
        y = _odd_strides(x.clone(), dim)
        assert torch.equal(serving.rotary(y, cos, sin, pos, out=y), want)

    qkv = torch.randn((b.tokens, 3 * 64), generator=g).to(dev)
    caches = []
    for odd in (False, True):
        k, v, *rest = b.device()
        q = serving.qk_rope_append_paged(qkv, cos, sin, *((_odd_strides(t, 1) if odd else t) for t in (k, v)), *rest, 1)
        caches.append((q, k.nan_to_num(9.0), v.nan_to_num(9.0)))
    assert all(torch.equal(x, y) for x, y in zip(*caches))


def test_a_cache_laid_out_position_by_position_of_one_kv_head(dev, path):
    """[n_pages, page, n_kv, D] turned into the pages' order: with one kv head contiguous() leaves it as it is."""
    b = ref.Batch([1, 2], [40, 70], 1, 128, 32, dev)
    k, v, *rest = b.device()
    q = torch.randn((b.tokens, 2, 128), generator=torch.Generator().manual_seed(1)).half().to(dev)
    want = serving.paged_attention(q, k, v, *rest, 2, 70, 0.1)
    turned = [torch.empty((t.shape[0], 32, 1, 128), dtype=t.dtype, device=dev).copy_(t.transpose(1, 2)).transpose(1, 2).contiguous()
              for t in (k, v)]
    assert turned[0].stride() != k.stride()
    assert torch.equal(serving.paged_attention(q, *turned, *rest, 2, 70, 0.1), want)


def test_outputs_between_the_rows_of_their_inputs(dev, path):
    """Memory of the same tensor that is none of the input's: queries inside wider rows with the output in the gap, keys
    turned into the values' place."""
    b = ref.Batch([1, 1], [40, 70], 2, 64, 16, dev)
    arrays = b.device()
    g = torch.Generator().manual_seed(1)
    wide = torch.randn((2, 12, 64), generator=g).half().to(dev)
    want = serving.paged_attention(wide[:, :2].contiguous(), *arrays, 1, 70, 0.1)
    out = wide.view(-1)[2 * 64:6 * 64].view(2, 2, 64)
    assert torch.equal(serving.paged_attention(wide[:, :2], *arrays, 1, 70, 0.1, out=out), want)
    cos, sin = (torch.from_numpy(t).to(dev) for t in serving.rope_table_scaled(64, 64, 1e4))
    pos = torch.arange(2, dtype=torch.int32, device=dev) + 9
    want = serving.rotary(wide[:, 6:8].contiguous(), cos, sin, pos)
    assert torch.equal(serving.rotary(wide[:, 6:8], cos, sin, pos, out=wide[:, 10:]), want)
    with pytest.raises(DttsError, match="shares memory"):
        serving.rotary(wide[:, 6:8], cos, sin, pos, out=wide[:, 7:9])
    with pytest.raises(DttsError, match="may not be the queries"):
        serving.paged_attention(wide[:, :2], *arrays, 1, 70, 0.1, out=wide.view(-1)[64:5 * 64].view(2, 2, 64))


def test_keys_and_values_side_by_side_in_one_pool(dev, path):
    """Pages of keys and of values in turn; the same tensor for both is refused."""
    b = ref.Batch([2, 1], [40, 70], 2, 64, 16, dev)
    k, v, *rest = b.device()
    pool = torch.stack([k, v], 1)
    cos, sin = (torch.from_numpy(t).to(dev) for t in serving.rope_table_scaled(128, 64, 1e4))
    qkv = torch.randn((b.tokens, 8 * 64), generator=torch.Generator().manual_seed(1)).half().to(dev)
    want = serving.qk_rope_append_paged(qkv, cos, sin, k, v, *rest, 4)
    got = serving.qk_rope_append_paged(qkv, cos, sin, pool[:, 0], pool[:, 1], *rest, 4)
    assert torch.equal(got, want)
    assert all(torch.equal(x.nan_to_num(9.0), y.nan_to_num(9.0)) for x, y in ((pool[:, 0], k), (pool[:, 1], v)))
    with pytest.raises(DttsError, match="share memory"):
        serving.qk_rope_append_paged(qkv, cos, sin, k, k, *rest, 4)


def test_starts_that_select_nothing_write_nothing(dev, path):
    """Starts that fall, lie outside the batch or are all alike: rows of `out` and slots of the cache that no sequence of
    theirs has stay as they were, bit for bit."""
    heads, c = 2, [30, 40, 50]
    b = ref.Batch([4, 3, 2], c, 2, 64, 16, dev, extra_tokens=2)
    cos, sin = (torch.from_numpy(t).to(dev) for t in serving.rope_table_scaled(64, 64, 1e4))
    qkv = torch.randn((b.tokens, (heads + 4) * 64), generator=torch.Generator().manual_seed(4)).half().to(dev)
    for starts, rows in (([9, 4, 2, 0], []), ([5, 3, -9, -9], []), ([100, 200, 300, 400], []), ([-8, -8, -8, 0], []),
                         ([11, 11, 11, 2 ** 31 - 1], []), ([6, 2, 2, 5], [2, 3, 4]), ([0, 0, 0, 3], [0, 1, 2]), ([3, 1, 4, 4], [1, 2, 3])):
        k, v, _, ctx, table = b.device()
        start = torch.tensor(starts, dtype=torch.int32, device=dev)
        k0, v0 = k.clone(), v.clone()
        out = torch.full((b.tokens, heads, 64), 9.0, dtype=torch.float16, device=dev)
        serving.qk_rope_append_paged(qkv, cos, sin, k, v, start, ctx, table, heads, out=out)
        assert bool((out[[t for t in range(b.tokens) if t not in rows]] == 9.0).all()), starts
        # positions that the selected rows have: sequence s's last n, where its starts rise
        slots = {(int(b.table[s, p // 16]), p % 16) for s in range(3) for p in range(max(0, c[s] - (starts[s + 1] - starts[s])), c[s])
                 if 0 <= starts[s] < starts[s + 1] <= b.tokens}
        kept = torch.ones(k.shape[0], 16, dtype=torch.bool)
        for at in slots:
            kept[at] = False
        for x, y in ((k, k0), (v, v0)):
            x, y = (t.transpose(1, 2)[kept.to(dev)] for t in (x, y))
            assert torch.equal(x.view(torch.int16), y.view(torch.int16)), starts
        out.fill_(9.0)
        for max_q, workspace in ((4, None), (200, torch.empty(0, dtype=torch.uint8, device=dev))):
            serving.paged_attention(qkv.view(b.tokens, heads + 4, 64)[:, :heads], k, v, start, ctx, table, max_q, 50, 0.1, out=out,
                                    workspace=workspace)
            assert bool((out[[t for t in range(b.tokens) if t not in rows]] == 9.0).all()), starts
