"""dtts_paged_attention_f16 over values that are not finite: they reach the tokens that see them, as the sum of the row says,
no others, and cost little more than finite ones."""
import numpy as np
import pytest
import torch

from dtts import serving

import _serving_ref as ref

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")

# (new tokens, contexts, heads, n_kv, head_dim, page, window): 16-row tiles of one and several tokens, 128-row ones, both in
# one batch, windows whose lower edge cuts a tile, contexts shorter than their chunk
BATCHES = [
    ([1, 1], [300, 50], 8, 2, 128, 16, 0),
    ([8, 5], [300, 70], 4, 1, 64, 16, 0),
    ([200], [500], 4, 1, 128, 64, 0),
    ([130, 1, 60], [400, 300, 60], 2, 2, 64, 32, 0),
    ([1, 8], [300, 300], 4, 1, 128, 16, 70),
    ([200, 1], [700, 90], 2, 1, 64, 64, 37),
    ([200, 8], [700, 300], 4, 2, 128, 16, 300),
    ([140, 3], [100, 2], 4, 2, 64, 16, 0),
]


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("n,c,heads,n_kv,hd,page,window", BATCHES)
def test_values_reach_who_sees_them(dev, n, c, heads, n_kv, hd, page, window, workspace):
    b = ref.Batch(n, c, n_kv, hd, page, dev, seed=len(n))
    g = torch.Generator().manual_seed(3)
    q = torch.randn((b.tokens, heads, hd), generator=g).half().to(dev)
    ws = None if workspace else torch.empty(0, dtype=torch.uint8, device=dev)

    def run(k, v):
        _, _, *rest = b.device()
        return serving.paged_attention(q, k, v, *rest, max(n), max(c), 0.1, window, workspace=ws).cpu().double()

    k, v, *_ = b.device()
    clean = run(k, v)
    hits = []  # (sequence, key, kv head, dimension, value): around the first token's own key, at a window's lower edge, far before
    for s, (m, x) in enumerate(zip(n, c)):
        first = x - m
        keys = [first - 40, first - 1, first, first + 1, first + m // 2, x - 1, first - window, first - window + 1, first - window + m // 2]
        for i, j in enumerate(keys):
            if 0 <= j < x:
                hits.append((s, j, i % n_kv, (7 * i + s) % hd, (NAN, INF, -INF)[i % 3]))
                if i % 2:
                    hits.append((s, j, i % n_kv, 5, INF if i % 4 == 1 else -INF))  # the same dimension: they meet
    for s, j, head, d, x in hits:
        v[b.table[s, j // page], head, j % page, d] = x
    got = run(k, v)
    # every weight is above 0: a row has the sum of what it sees that is not finite, and is as it was elsewhere
    add = torch.zeros_like(got)
    seen_by = heads // n_kv
    cells = {}
    for s, j, head, d, x in hits:
        cells[s, j, head, d] = x  # the last one written
    for (s, j, head, d), x in cells.items():
        for t in range(n[s]):
            pos = c[s] - n[s] + t
            if j <= pos and (not window or j > pos - window):
                add[int(b.start[s]) + t, head * seen_by:(head + 1) * seen_by, d] += x
    spoilt = ~torch.isfinite(add)
    assert bool(spoilt.any()) and torch.equal(got[~spoilt], clean[~spoilt])
    assert torch.equal(got[spoilt].nan_to_num(9.0, 7.0, 8.0), add[spoilt].nan_to_num(9.0, 7.0, 8.0))


@pytest.mark.parametrize("n,heads", [(100, 4), (1, 4), (8, 4)])
@pytest.mark.parametrize("where", [3, -1])
def test_a_value_that_is_not_finite_costs_little(dev, n, heads, where):
    """A long context with one NaN, which every token sees or the last one alone: within a few times the time of finite
    values (a row taken again key by key has 6000 steps of a trip to memory each)."""
    c = 6000
    b = ref.Batch([n], [c], 1, 128, 16, dev)
    arrays = b.device()
    q = torch.randn((n, heads, 128), generator=torch.Generator().manual_seed(1)).half().to(dev)

    def best():
        times = []
        for _ in range(6):
            e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            e[0].record()
            out = serving.paged_attention(q, *arrays, n, c, 0.1)
            e[1].record()
            torch.cuda.synchronize()
            times.append(e[0].elapsed_time(e[1]) * 1e3)
        return min(times), out

    clean, _ = best()
    at = where % c
    arrays[1][b.table[0, at // 16], 0, at % 16, 7] = NAN
    bad, out = best()
    seen = torch.isnan(out[:, :, 7]).all(1).cpu().numpy()
    assert np.array_equal(seen, np.arange(c - n, c) >= at)
    assert bad <= 5 * clean + 100, (bad, clean)
