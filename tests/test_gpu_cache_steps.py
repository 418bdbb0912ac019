"""The cache's calls together, as a server makes them: prompts, beams that fork and part, streams that run past their windows, a pool
that is compacted between steps. Every step's attention is held to a 64-bit evaluation of a cache kept row by row on the host."""
import numpy as np
import pytest
import torch

from dtts import serving

import _pages_ref as ref

pytestmark = pytest.mark.gpu


class Host:
    """What every sequence has cached, position by position, as the f16 values that its pages stand for."""

    def __init__(self, b):
        self.k, self.v = [[] for _ in range(b)], [[] for _ in range(b)]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("hd", [64, 128])
def test_a_server(dev, bits, hd):
    b, m, page, n_pages, heads, n_kv, window, sinks, layers = 6, 24, 16, 90, 4, 2, 100, 5, 2
    rng = np.random.RandomState(bits + hd)
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    table, refs = torch.full((b, m), -1, dtype=torch.int32, device=dev), torch.zeros(n_pages, dtype=torch.int32, device=dev)
    shape, dtype = ((n_pages, n_kv, page, hd), torch.float16) if bits == 16 else ((n_pages, n_kv, page, 5 * hd // 8), torch.uint8)
    pools = [[torch.zeros(shape, dtype=dtype, device=dev) for _ in range(2)] for _ in range(layers)]
    if bits == 4:
        for k, v in pools:  # nothing that was never written may count
            k.fill_(255), v.fill_(255)
    cos, sin = (torch.from_numpy(t).to(dev) for t in serving.rope_table_scaled(m * page, hd, 1e4))
    lengths, cached = np.zeros(b, int), [[[] for _ in range(b)] for _ in range(layers)]
    script = ["prompts", "beams"] + ["decode"] * 3 + ["beams"] + ["decode"] * 20 + ["end", "compact"] + ["decode"] * 4 + \
        ["prompts", "beams", "compact"] + ["decode"] * 18
    for kind in script:
        if kind == "compact":
            src, dst, used = serving.compact_pages(table, refs)
            for pool in pools:
                serving.copy_pages(pool, src, dst)
            assert int(used) == int((refs > 0).sum()) and bool((refs[:int(used)] > 0).all())
            continue
        if kind in ("beams", "end"):
            live = np.nonzero(lengths)[0]
            parent = rng.choice(live, b) if kind == "beams" else np.where(np.arange(b) % 2, np.arange(b), -1)
            if rng.rand() < 0.5:
                serving.fork_pages(table, refs, i32(parent), out=table)
            else:
                table = serving.fork_pages(table, refs, i32(parent))
            for layer in range(layers):
                cached[layer] = [list(cached[layer][p]) if p >= 0 else [] for p in parent]
            lengths = np.where(parent >= 0, lengths[parent], 0)
            continue
        n = np.where(lengths > 0, 1, 0)
        if kind == "prompts":
            n = np.where(lengths == 0, rng.choice([0, 3, 37, 70], b), 1)
            n[0] = n[0] or 5
        lengths = lengths + n
        start, ctx = i32(np.concatenate([[0], np.cumsum(n)])), i32(lengths)
        src, dst, lacking = serving.claim_pages(table, refs, start, ctx, page)
        assert int(lacking) == 0
        tokens = int(n.sum())
        for layer, pool in enumerate(pools):
            serving.copy_pages(pool, src, dst)
            qkv = torch.from_numpy(rng.randn(tokens, (heads + 2 * n_kv) * hd)).float().to(dev)
            q = serving.qk_rope_append_paged(qkv, cos, sin, *pool, start, ctx, table, heads)
            out = serving.paged_attention(q, *pool, start, ctx, table, int(n.max()), int(lengths.max()), hd ** -0.5, window, sinks=sinks)
            f16 = pool if bits == 16 else serving.unpack_pages(*pool)
            k, v, rows = *(t.cpu() for t in f16), table.cpu().numpy()
            at, want_rows = 0, []
            for s in range(b):
                for i in range(n[s]):
                    p = lengths[s] - n[s] + i
                    cached[layer][s].append(tuple(t[rows[s, p // page], :, p % page].clone() for t in (k, v)))
                at += n[s]
            # each sequence as one page of its own, from what was cached when it was written
            longest = max(page, 1 << int(lengths.max() - 1).bit_length())
            own = [torch.zeros((b, n_kv, longest, hd), dtype=torch.float16) for _ in range(2)]
            for s in range(b):
                for p, pair in enumerate(cached[layer][s]):
                    for t, x in zip(own, pair):
                        t[s, :, p] = x
            want, bound = ref.attention(q, *own, np.concatenate([[0], np.cumsum(n)]), lengths, np.arange(b)[:, None], longest, hd ** -0.5,
                                        window, sinks)
            err = (out.cpu().double() - want).abs()
            assert bool((err <= bound).all()), (kind, layer, float((err / bound).max()))
        serving.trim_pages(table, refs, ctx, page, window, sinks)
        held = table[table >= 0].cpu().numpy()
        assert np.array_equal(np.bincount(held, minlength=n_pages), refs.cpu().numpy())
