"""The serving ops in 64 bits, written from their definitions, and ragged paged batches to run them on."""
import numpy as np
import torch


def turn(x, cos, sin, interleaved):
    """x [n, heads, D] f64 with its first 2 * cos.shape[1] dimensions turned by cos, sin [n, rot / 2]; and the
    magnitude |x1 c| + |x2 s| that a product's rounding is relative to."""
    h = cos.shape[1]
    c, s = cos[:, None], sin[:, None]
    y, mag = x.copy(), np.abs(x)
    a, b = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if interleaved else (x[..., :h], x[..., h:2 * h])
    o = (a * c - b * s, b * c + a * s), (np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s))
    for dst, (p, q) in zip((y, mag), o):
        if interleaved:
            dst[..., 0:2 * h:2], dst[..., 1:2 * h:2] = p, q
        else:
            dst[..., :h], dst[..., h:2 * h] = p, q
    return y, mag


def rms(x, w, eps):
    return x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * w


class Batch:
    """Sequences of n[i] new tokens and context c[i] over pages scattered in a pool: every slot that holds no
    position of a sequence is NaN, table entries past a sequence's last page are -1."""

    def __init__(self, n, c, n_kv, head_dim, page, dev, seed=0, extra_tokens=0, stride_pages=1, spare=2):
        rng = np.random.RandomState(seed)
        self.n, self.c, self.n_kv, self.hd, self.page, self.dev = list(n), list(c), n_kv, head_dim, page, dev
        need = [-(-max(x, 0) // page) for x in c]
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages)
        table = np.full((len(n), max(max(need), 1)), -1, np.int32)
        at = 0
        for i, k in enumerate(need):
            table[i, :k] = order[at:at + k]
            at += k
        self.table = table
        self.start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        self.tokens = int(self.start[-1]) + extra_tokens
        g = torch.Generator().manual_seed(seed)
        shape = (self.n_pages * stride_pages, n_kv, page, head_dim)
        self.k, self.v = (torch.full(shape, float("nan"), dtype=torch.float16)[::stride_pages] for _ in range(2))
        for i, x in enumerate(c):
            for p in range(need[i]):
                m = min(page, x - p * page)
                for t, s in ((self.k, 1.3), (self.v, 1.0)):
                    t[table[i, p], :, :m] = (torch.randn((n_kv, m, head_dim), generator=g) * s).half()

    def device(self):
        def up(a):
            return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(self.dev)

        k, v = (torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=self.dev).copy_(t) for t in (self.k, self.v))
        return k, v, up(self.start), up(self.c), up(self.table)


def attention(q, k, v, start, context, table, page, scale, window):
    """(out, bound) f64 on the CPU. q [tokens, heads, D]; bound: how far the kernel may be off, from the
    roundings it makes (2^-24 in f32, 2^-11 of each weight and of the output in f16)."""
    q, k, v = (t.cpu() for t in (q, k, v))
    heads, hd = q.shape[1:]
    g = heads // k.shape[1]
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for s in range(len(context)):
        a, e, c = int(start[s]), int(start[s + 1]), int(context[s])
        n = e - a
        keys = [j for j in range(max(0, min(c, table.shape[1] * page))) if 0 <= table[s, j // page] < k.shape[0]]
        if n == 0 or not keys:
            continue
        j = torch.tensor(keys)
        ids, slot = torch.from_numpy(table[s].astype(np.int64))[j // page], j % page
        ks, vs = k[ids, :, slot].double(), v[ids, :, slot].double()  # [keys, n_kv, D]
        pos = torch.arange(c - n, c)[:, None]
        seen = (j <= pos) & (j > pos - window if window else j >= 0)
        for h in range(heads):
            kk, vv = ks[:, h // g], vs[:, h // g]
            qq = q[a:e, h].double()
            z = (qq @ kk.T * scale).masked_fill(~seen, -np.inf)
            m = z.amax(-1, keepdim=True).clamp(min=-1e300)
            p = (z - m).exp()
            l = p.sum(-1, keepdim=True)
            none = ~seen.any(-1, keepdim=True)
            p = torch.where(none, 0.0, p / l)
            # a masked value counts for nothing, whatever it is
            rows = [p[i][seen[i]] @ vv[seen[i]] if seen[i].any() else torch.zeros(hd, dtype=torch.float64) for i in range(n)] \
                if not torch.isfinite(vv).all() else list(p @ vv)
            o = torch.stack(rows)
            pv = p @ vv.nan_to_num(0, 0, 0).abs()
            # scores: hd products summed in f32; weights: e^x of a score that far off, one ulp, and f16; sums. A
            # score's error is |scale| times its dot's, whatever the sign: |scale a - scale b| = |scale| |a - b|
            dots = (qq.nan_to_num(0, 0, 0).abs() @ kk.nan_to_num(0, 0, 0).abs().T).amax(-1, keepdim=True) * abs(scale)
            rel = 2 * (hd + 4) * 2.0 ** -24 * dots + (len(keys) / 16 + 32) * 2.0 ** -24
            far = len(keys) * 2.0 ** -25 / l.clamp(min=1.0) * vv.nan_to_num(0, 0, 0).abs().amax()  # weights under f16's normal range
            out[a:e, h] = o
            bound[a:e, h] = 2.0 ** -11 * (o.abs() + pv) + rel * (pv + o.abs()) + far + 2.0 ** -25
    return out, bound


def sample(x, u, t, k, p, m):
    """One row, x f64: (token, log-probability)."""
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    if top == -np.inf:
        return -1, -np.inf
    if not t > 0:
        return int(order[0]), 0.0
    w = np.zeros_like(x)
    if top == np.inf:
        w[x == top] = 1.0
    else:
        w = np.exp((x - top) / t)
    ws = w[order]
    rank = np.arange(len(x))
    kk = k if 0 < k < len(x) else len(x)
    ws = np.where((rank < kk) & (x[order] > -np.inf), ws, 0.0)
    c = np.cumsum(ws)
    before = np.concatenate([[0], c[:-1]])
    keep = (rank < kk) & ((before < p * c[-1]) | (not p < 1)) & ((ws >= m) | (not m > 0)) | (rank == 0)
    wk = np.zeros_like(w)
    wk[order[keep]] = ws[keep]
    c = np.cumsum(wk)
    u = min(max(u, 0.0), 1 - 2.0 ** -53) if u == u else 0.0
    i = int(np.searchsorted(c, u * c[-1], side="right"))
    i = min(i, int(np.max(np.nonzero(wk)[0])))
    return i, float((0.0 if x[i] == top else (x[i] - top) / t) - np.log(c[-1]))
