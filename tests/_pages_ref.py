"""Pages in 4 bits, windows with sinks and the page calls, from their definitions: numpy and plain loops."""
import numpy as np
import torch


# ---------------------------------------------------------------- 4-bit pages

def quantise(x):
    """Rows [.., D] f64 as (n, d, b): the 4-bit numbers, and the pairs [.., D / 32] as the f16 numbers they are."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        lo, hi = g.min(-1), g.max(-1)
        d = ((hi - lo) / 15).astype(np.float16)
        b = (lo - 64 * d.astype(np.float64)).astype(np.float16)
        d64, b64 = d.astype(np.float64), b.astype(np.float64)
        ends = np.stack([64 * d64 + b64, 79 * d64 + b64]).astype(np.float16)
        bad = ~np.isfinite(ends).all(0) | ~np.isfinite(g).all(-1)
        d, b = np.where(bad, np.float16(np.nan), d), np.where(bad, np.float16(np.nan), b)
        t = (g - (64 * d64 + b64)[..., None]) / np.where(d64 > 0, d64, 1.0)[..., None]
        n = np.where((d64 > 0)[..., None] & ~bad[..., None], np.clip(np.rint(np.nan_to_num(t)), 0, 15), 0)
    return n.astype(np.int64).reshape(x.shape), d, b


def pack(x, values):
    """Pages [n, n_kv, page, D] f64 as uint8 [n, n_kv, page, 5 D / 8]."""
    n, n_kv, page, hd = x.shape
    codes, d, b = quantise(x)
    codes = codes.reshape(n, n_kv, page, hd // 8, 8).astype(np.uint32)
    words = np.zeros(codes.shape[:-1], np.uint32)
    for e in range(8):
        words |= codes[..., e] << np.uint32(4 * (e // 2) + 16 * (e % 2))
    if values:
        words = words.reshape(n, n_kv, page // 4, 4, hd // 8).swapaxes(-1, -2)
    pairs = np.stack([d, b], -1).transpose(0, 1, 3, 2, 4)  # [n, n_kv, D / 32, page, 2]
    flat = [np.ascontiguousarray(t).view(np.uint8).reshape(n, n_kv, -1) for t in (words, pairs)]
    return np.concatenate(flat, -1).reshape(n, n_kv, page, 5 * hd // 8)


def unpack(pages, values):
    """uint8 pages as (values f64, d, b): the values are f16 numbers, d and b [n, n_kv, page, D / 32]."""
    n, n_kv, page, row = pages.shape
    hd = row * 8 // 5
    flat = pages.reshape(n, n_kv, -1)
    words = np.ascontiguousarray(flat[..., :page * hd // 2]).view(np.uint32)
    words = words.reshape(n, n_kv, page // 4, hd // 8, 4).swapaxes(-1, -2) if values else words
    words = words.reshape(n, n_kv, page, hd // 8)
    codes = np.stack([words >> np.uint32(4 * (e // 2) + 16 * (e % 2)) & np.uint32(15) for e in range(8)], -1)
    pairs = np.ascontiguousarray(flat[..., page * hd // 2:]).view(np.float16).reshape(n, n_kv, hd // 32, page, 2)
    d, b = (pairs[..., i].transpose(0, 1, 3, 2).astype(np.float64) for i in (0, 1))
    with np.errstate(all="ignore"):
        x = (64.0 + codes.reshape(n, n_kv, page, hd // 32, 32)) * d[..., None] + b[..., None]
        return x.astype(np.float16).astype(np.float64).reshape(n, n_kv, page, hd), d, b


def repack(t, values, stride_pages=1):
    """f16 pages as 4-bit ones on the CPU, torch uint8 (with gaps between the pages, where asked)."""
    p = torch.from_numpy(pack(t.double().numpy(), values))
    if stride_pages == 1:
        return p
    wide = torch.full((p.shape[0] * stride_pages, *p.shape[1:]), 255, dtype=torch.uint8)
    wide[::stride_pages] = p
    return wide[::stride_pages]


# ---------------------------------------------------------------- attention

def attention(q, k, v, start, context, table, page, scale, window, sinks=0):
    """(out, bound) f64 on the CPU over f16 pages k, v: see attention in _serving_ref, with the first `sinks` positions seen too. The
    bound counts the kernel's roundings: 2^-24 a step in f32, 2^-11 of each weight and of the output in f16."""
    q, k, v = (t.cpu().double() for t in (q, k, v))
    heads, hd = q.shape[1:]
    g = heads // k.shape[1]
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for s, c in enumerate(context):
        a, e, c = int(start[s]), int(start[s + 1]), int(c)
        held = [j for j in range(max(0, min(c, table.shape[1] * page))) if 0 <= table[s, j // page] < k.shape[0]]
        for t in range(a, e):
            p = c - (e - a) + t - a
            seen = torch.tensor([j for j in held if j <= p and (not window or j > p - window or j < sinks)], dtype=torch.long)
            if not len(seen):
                continue
            ids, slot = torch.from_numpy(table[s].astype(np.int64))[seen // page], seen % page
            ks, vs = k[ids, :, slot].repeat_interleave(g, 1), v[ids, :, slot].repeat_interleave(g, 1)  # [keys, heads, D]
            z = (q[t] * ks).sum(-1) * scale
            w = (z - z.amax(0)).exp()
            l = w.sum(0)
            w = (w / l)[..., None]
            o, pv = (w * vs).sum(0), (w * vs.nan_to_num(0, 0, 0).abs()).sum(0)
            dots = (q[t].abs() * ks.abs()).sum(-1).amax(0)[:, None] * abs(scale)
            rel = 2 * (hd + 4) * 2.0 ** -24 * dots + (len(seen) / 16 + 32) * 2.0 ** -24
            far = len(seen) * 2.0 ** -25 / l.clamp(min=1.0)[:, None] * vs.nan_to_num(0, 0, 0).abs().amax()
            out[t] = o
            bound[t] = 2.0 ** -11 * (o.abs() + pv) + rel * (pv + o.abs()) + far + 2.0 ** -25
    return out, bound


# ---------------------------------------------------------------- pages

def fork(table, refs, parent):
    table, refs = table.copy(), refs.copy()
    new = np.full((len(parent), table.shape[1]), -1, np.int32)
    for i, p in enumerate(parent):
        if 0 <= p < len(table):
            new[i] = table[p]
    for t, by in ((new, 1), (table, -1)):
        for e in t.flatten():
            if 0 <= e < len(refs):
                refs[e] += by
    return new, refs


def claim(table, refs, q_start, context, page):
    """One writer after another. A page that loses an owner never gets free here, so what is free is so from the start."""
    new, counts = table.copy(), refs.copy()
    b, m = table.shape
    src, dst = np.full(b, -1, np.int32), np.full(b, -1, np.int32)
    free = [p for p in range(len(refs)) if refs[p] < 1]
    need = 0
    for s in range(b):
        n = max(0, int(q_start[s + 1]) - int(q_start[s]))
        c = max(0, int(context[s]))
        at = max(0, c - n)
        for j in range(m):
            if n == 0 or j < at // page or j * page >= min(c, m * page) or at >= min(c, m * page):
                continue
            e = int(table[s, j])
            held = 0 <= e < len(refs) and refs[e] > 0
            if held and counts[e] == 1:
                continue
            if held:
                counts[e] -= 1
            if need < len(free):
                p = free[need]
                new[s, j], counts[p] = p, 1
                if held and j == at // page and at % page:
                    src[s], dst[s] = e, p
            need += 1
    if need > len(free):
        none = np.full(b, -1, np.int32)
        return table.copy(), refs.copy(), none, none.copy(), need - len(free)
    return new, counts, src, dst, 0


def trim(table, refs, context, page, window, sinks):
    table, refs = table.copy(), refs.copy()
    for s, c in enumerate(context):
        for j in range(table.shape[1]):
            if j * page >= sinks and (j + 1) * page <= c - window + 1:
                if 0 <= table[s, j] < len(refs):
                    refs[table[s, j]] -= 1
                table[s, j] = -1
    return table, refs


def compact(table, refs):
    used = [p for p in range(len(refs)) if refs[p] > 0]
    movers, holes = [p for p in used if p >= len(used)], [p for p in range(len(used)) if refs[p] < 1]
    to = {p: p for p in used} | dict(zip(movers, holes))
    src, dst = np.full(len(refs), -1, np.int32), np.full(len(refs), -1, np.int32)
    src[:len(movers)], dst[:len(holes)] = movers, holes
    counts = np.zeros_like(refs)
    for p in used:
        counts[to[p]] = refs[p]
    return np.vectorize(lambda e: to.get(int(e), -1), otypes=[np.int32])(table).reshape(table.shape), counts, src, dst, len(used)
