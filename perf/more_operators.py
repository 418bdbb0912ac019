"""Operators of a server's cache, as measurable cases: 4-bit pages, windows with sinks, pages that are
forked, claimed, trimmed, compacted and copied.

A case is a dict of plain values; ``kind`` says which operators it goes through:

  attention  attention of each sequence's new tokens over 4-bit pages, or over f16 ones with a sliding
             window beside the first tokens (``dtts.serving.paged_attention``)
  append     QK-norm, rotary positions and the write into 4-bit pages, whose values are then read back
             (``dtts.serving.qk_rope_append_paged``, ``unpack_pages``)
  fork       a step of beams: rows take their parents' pages, claim what they write next, and copy what
             they share (``fork_pages``, ``claim_pages``, ``copy_pages``)
  compact    pages that no window reaches are freed, the others moved together (``trim_pages``,
             ``compact_pages``, ``copy_pages``)

Lengths and page tables of a case follow from the case alone; values follow from the seed.

A 4-bit page of a kv head holds `page` rows of D values in groups of 32: value = f16(c d + b), c = 64 + n, n the
group member's 4 bits, d and b the group's f16 pair. First the rows' bits, D / 8 words of 32 a row: element 8 w + 2 i
of a row in bits 4 i of its word w, element 8 w + 2 i + 1 in bits 16 + 4 i; the keys' words in the order [row][w], the
values' in the order [row / 4][w][row % 4]. Then the pairs, [D / 32][row].
"""
from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda:0"
F16, F32, F64, I32 = torch.float16, torch.float32, torch.float64, torch.int32


def listed():
    return [
        # one request, one token, a short context: the smallest call
        dict(name="attention4_1x1_300", kind="attention", bits=4, b=1, prefills=0, q=1, ctx=300, heads=16, n_kv=8,
             head_dim=128, page=16, window=0, sinks=0, lens=21),
        # a talker's batch, every lane at its own position
        dict(name="attention4_48x1_1536", kind="attention", bits=4, b=48, prefills=0, q=1, ctx=1536, heads=16, n_kv=8,
             head_dim=128, page=16, window=0, sinks=0, lens=22),
        # few requests with very long contexts, what 4 bits are for: eight query heads a kv head
        dict(name="attention4_5x1_65000", kind="attention", bits=4, b=5, prefills=0, q=1, ctx=65000, heads=32, n_kv=4,
             head_dim=128, page=64, window=0, sinks=0, lens=23),
        # a long prompt's chunk after what is already cached
        dict(name="attention4_1x1025_7000", kind="attention", bits=4, b=1, prefills=1, q=1025, ctx=7000, heads=32, n_kv=8,
             head_dim=128, page=64, window=0, sinks=0, lens=24),
        # streams that run on: a window and four first tokens, over f16 pages that are freed between them
        dict(name="sinks_64x1_20001", kind="attention", bits=16, b=64, prefills=0, q=1, ctx=20001, heads=32, n_kv=4,
             head_dim=64, page=32, window=2048, sinks=4, lens=25),
        # prompts' chunks beside decoding streams, a long visible prefix, in 4 bits
        dict(name="sinks4_mixed_9", kind="attention", bits=4, b=9, prefills=2, q=700, ctx=6001, heads=16, n_kv=2,
             head_dim=128, page=64, window=1000, sinks=130, lens=26),
        # a talker's decode step: one f32 row of q, k and v per lane, with QK-norm
        dict(name="append4_decode_48", kind="append", dtype="f32", b=48, prefills=0, q=1, ctx=400, heads=16, n_kv=8,
             head_dim=128, rot=128, interleaved=False, norm=True, page=16, lens=27),
        # prompts of several requests at once, f16 rows, half of a 64-wide head rotated in interleaved pairs
        dict(name="append4_prefill_5", kind="append", dtype="f16", b=5, prefills=5, q=1201, ctx=1600, heads=16, n_kv=8,
             head_dim=64, rot=32, interleaved=True, norm=False, page=64, lens=28),
        # four samples of one request after its prompt, over a small pool
        dict(name="fork_1x4", kind="fork", groups=1, beams=4, ctx=301, page=16, pool=200, n_kv=8, head_dim=128, bits=16, lens=29),
        # beams of a batch, reordered within their request, ended ones among them, in 4 bits
        dict(name="fork_40x4", kind="fork", groups=40, beams=4, ctx=3001, page=32, pool=20011, n_kv=4, head_dim=128, bits=4, lens=30),
        # a pool half of whose pages ended requests and windows have left, of f16 keys and values
        dict(name="compact_6000", kind="compact", b=61, ctx=2999, page=32, pool=6001, n_kv=8, head_dim=64, bits=16, window=1024,
             sinks=4, lens=31),
        # a large pool of small 4-bit pages
        dict(name="compact_100000", kind="compact", b=200, ctx=8001, page=16, pool=100003, n_kv=2, head_dim=64, bits=4, window=4096,
             sinks=100, lens=32),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "attention", "append", "fork", "compact"])
    hd, bits = rng.choice([64, 128, 128]), rng.choice([4, 16])
    if kind == "fork":
        groups, beams, page = _log_int(rng, 1, 60), rng.choice([2, 3, 4, 8]), rng.choice([16, 32, 64])
        ctx = _log_int(rng, 2, 6000)
        pool = groups * (-(-ctx // page) + beams * (64 // page + 2)) + _log_int(rng, 1, 4000)
        return dict(kind=kind, groups=groups, beams=beams, ctx=ctx, page=page, pool=pool, n_kv=rng.choice([1, 2, 4]), head_dim=hd,
                    bits=bits, lens=rng.randrange(1 << 20))
    if kind == "compact":
        b, page = _log_int(rng, 1, 200), rng.choice([16, 32, 64])
        ctx = _log_int(rng, page, 6000)
        return dict(kind=kind, b=b, ctx=ctx, page=page, pool=b * -(-ctx // page) + _log_int(rng, 1, 4000), n_kv=rng.choice([1, 2, 4]),
                    head_dim=hd, bits=4 if b * ctx > 100000 else bits, window=_log_int(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 64]),
                    lens=rng.randrange(1 << 20))
    n_kv = rng.choice([1, 2, 4, 8, 16])
    heads = n_kv * rng.choice([1, 2, 4, 5, 8] if n_kv < 8 else [1, 2, 4])
    page = rng.choice([16, 32, 64, 128])
    mix = rng.choice(["decode", "decode", "prefill", "mixed"])
    b = _log_int(rng, 1, {"decode": 96, "prefill": 8, "mixed": 48}[mix])
    q = 1 if mix == "decode" else _log_int(rng, 2, 1500 // (b if mix == "prefill" else 1))
    prefills = 0 if mix == "decode" else b if mix == "prefill" else rng.randint(1, max(1, b // 8))
    case = dict(kind=kind, b=b, prefills=prefills, q=q, heads=heads, n_kv=n_kv, head_dim=hd, page=page,
                lens=rng.randrange(1 << 20))
    if kind == "append":
        return dict(case, dtype=rng.choice(["f32", "f16"]), ctx=q + _log_int(rng, 1, 600), norm=rng.random() < 0.5,
                    rot=rng.choice([hd, hd, hd // 2]), interleaved=rng.random() < 0.3)
    most = min(66000, int(4e8) // (b * q * heads), int(4e9) // (b * n_kv * hd * 8))
    window = _log_int(rng, 16, 4096) if bits == 16 else rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
    sinks = rng.choice([1, 4, 4, 16, 130]) if bits == 16 or window and rng.random() < 0.5 else 0
    return dict(case, bits=bits, ctx=q + _log_int(rng, 1, max(2, most - q)), window=window, sinks=sinks)


# ---------------------------------------------------------------- inputs from the seed alone

class _Draw:
    """torch's generator on the device, one stream per seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def normal(self, shape, std=1.0):
        return torch.randn(shape, generator=self.g, device=DEV) * std

    def uniform(self, shape, lo, hi):
        return torch.rand(shape, generator=self.g, device=DEV) * (hi - lo) + lo

    def bytes(self, shape):
        return torch.randint(0, 256, shape, generator=self.g, device=DEV, dtype=torch.uint8)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def _cache(d, bits, pool, n_kv, page, hd, std):
    """Pages as earlier steps left them: normal values, or in 4 bits any codes between a group's least and largest."""
    if bits == 16:
        return (d.normal((pool, n_kv, page, hd)) * std).half()
    step = d.uniform((pool, n_kv, hd // 32, page), 0.7, 1.3).mul_(0.25 * std).half()
    least = d.uniform(step.shape, -2.5, -1.5).mul_(std)
    pairs = torch.stack([step, (least - 64 * step.float()).half()], -1)
    codes = d.bytes((pool, n_kv, page * hd // 2))
    return torch.cat([codes, pairs.view(torch.uint8).view(pool, n_kv, -1)], -1).view(pool, n_kv, page, 5 * hd // 8)


def _tables(length, rot):
    f = 1e6 ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    a = torch.arange(length, device=DEV, dtype=F64)[:, None] * torch.from_numpy(f).to(DEV)[None]
    return a.cos().float(), a.sin().float()


def _lengths(case):
    """Each sequence's new tokens and context (new ones included). The first has the largest of both; with
    four or more, one decoding slot is idle."""
    rng, n, c = random.Random(case["lens"]), [], []
    for i in range(case["b"]):
        chunk = i < case["prefills"]
        n.append(case["q"] if i == 0 else rng.randint(max(1, case["q"] // 3), case["q"]) if chunk else 1)
        c.append(case["ctx"] if i == 0 else rng.randint(n[-1], case["ctx"]))
    if case["b"] >= 4 and not case["prefills"] == case["b"]:
        n[case["b"] // 2 if case["prefills"] <= case["b"] // 2 else -1] = 0
    return n, c


def _batch(case):
    """q_start, contexts and the page table of a ragged batch: its pages scattered over a pool, -1 past a
    sequence's last and where its window has left the page (but for the first tokens')."""
    n, c = _lengths(case)
    page, window, sinks = case["page"], case.get("window", 0), case.get("sinks", 0)
    counts = [-(-x // page) for x in c]
    held = [[j for j in range(k) if not window or j * page < sinks or (j + 1) * page > x - y - window + 1]
            for k, x, y in zip(counts, c, n)]
    pool = sum(map(len, held)) + 3
    order = np.random.RandomState(case["lens"]).permutation(pool)
    table = np.full((case["b"], max(counts)), -1, np.int32)
    at = 0
    for i, blocks in enumerate(held):
        table[i, blocks] = order[at:at + len(blocks)]
        at += len(blocks)
    start = np.concatenate([[0], np.cumsum(n)])
    return dict(q_start=_dev(start), context=_dev(c), pages=_dev(table), tokens=int(start[-1]), pool=pool)


def _beams(case):
    """The tables of a step that has chosen its beams: each request's beams share their prompt's pages and own what they
    have written since, 64 tokens at most; then the parents, one in seven rows ended, and the contexts with the next token."""
    rng = random.Random(case["lens"])
    page, beams, b = case["page"], case["beams"], case["groups"] * case["beams"]
    longest = -(-case["ctx"] // page) + 2
    ids = np.random.RandomState(case["lens"]).permutation(case["pool"])
    table, refs = np.full((b, longest), -1, np.int32), np.zeros(case["pool"], np.int32)
    lengths, at = [], 0
    for g in range(case["groups"]):
        n = case["ctx"] if g == 0 else rng.randint(1, case["ctx"])
        shared = max(0, n - rng.randint(0, 64)) // page  # what it had before it had beams
        for i in range(beams):
            s = g * beams + i
            for j in range(-(-n // page)):
                if j < shared and i > 0:
                    table[s, j] = table[g * beams, j]
                else:
                    table[s, j] = ids[at]
                    at += 1
                refs[table[s, j]] += 1
            lengths.append(n)
    parent = np.array([s - s % beams + rng.randrange(beams) for s in range(b)], np.int32)
    for s in range(b):
        if s % 7 == 6:
            parent[s] = -1
    live = parent >= 0
    context = np.where(live, np.array(lengths)[parent] + 1, 0)
    return dict(pages=_dev(table), refs=_dev(refs), parent=_dev(parent), context=_dev(context),
                q_start=_dev(np.concatenate([[0], np.cumsum(live)])))


def _fragments(case):
    """A pool after a while: sequences' pages at random places, a third of the sequences ended."""
    rng = random.Random(case["lens"])
    page, longest = case["page"], -(-case["ctx"] // case["page"])
    ids = np.random.RandomState(case["lens"]).permutation(case["pool"])
    table, refs = np.full((case["b"], longest), -1, np.int32), np.zeros(case["pool"], np.int32)
    context, at = [], 0
    for s in range(case["b"]):
        c = case["ctx"] if s == 0 else rng.randint(1, case["ctx"])
        k = -(-c // page)
        if s % 3 == 2:
            c = 0
        else:
            table[s, :k] = ids[at:at + k]
            refs[table[s, :k]] = 1
        at += k
        context.append(c)
    return dict(pages=_dev(table), refs=_dev(refs), context=_dev(context))


def prepare(case, seed):
    d, kind = _Draw(seed), case["kind"]
    if kind in ("fork", "compact"):
        s = dict(case=case, **(_beams if kind == "fork" else _fragments)(case))
        s["k"], s["v"] = (_cache(d, case["bits"], case["pool"], case["n_kv"], case["page"], case["head_dim"], x) for x in (1.3, 1.0))
        return s
    s = dict(case=case, **_batch(case))
    s["k"], s["v"] = (_cache(d, case.get("bits", 4), s["pool"], case["n_kv"], case["page"], case["head_dim"], x) for x in (1.3, 1.0))
    if kind == "attention":
        s["q"] = d.normal((s["tokens"], case["heads"], case["head_dim"]), 1.3).half()
        return s
    qkv = d.normal((s["tokens"], (case["heads"] + 2 * case["n_kv"]) * case["head_dim"]))
    s["qkv"] = qkv.half() if case["dtype"] == "f16" else qkv
    s["cos"], s["sin"] = _tables(case["ctx"], case["rot"])
    s["norms"] = d.uniform((2, case["head_dim"]), 0.8, 1.2) if case["norm"] else None
    return s


# ---------------------------------------------------------------- the plain forms: 4-bit pages

SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)


def _unpack(pages, values):
    """The f16 values [n, n_kv, page, D] that 4-bit pages stand for."""
    n, n_kv, page = pages.shape[:3]
    hd = pages.shape[3] * 8 // 5
    flat = pages.reshape(n, n_kv, -1)
    words = flat[..., :page * hd // 2].contiguous().view(I32)
    if values:
        words = words.view(n, n_kv, page // 4, hd // 8, 4).transpose(-1, -2)
    codes = (words.reshape(n, n_kv, page, hd // 8, 1) >> torch.tensor(SHIFTS, device=DEV, dtype=I32)) & 15
    pairs = flat[..., page * hd // 2:].contiguous().view(F16).view(n, n_kv, hd // 32, page, 2).float()
    step, base = (pairs[..., i].transpose(-1, -2).repeat_interleave(32, -1) for i in (0, 1))
    return ((64.0 + codes.view(n, n_kv, page, hd)) * step + base).half()


def _quantise(x):
    """Rows [.., D] f64 as (codes 0 .. 15, step, base), the last two [.., D / 32] f16."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    least, most = g.amin(-1), g.amax(-1)
    step = ((most - least) / 15).half()
    base = (least - 64 * step.double()).half()
    at = (g - base.double()[..., None]) / step.double()[..., None] - 64
    return torch.where(step[..., None] == 0, 0.0, at).round().clamp(0, 15).to(I32).view(x.shape), step, base


def _write(pages, values, x, ids, slot):
    """Rows x [tokens, n_kv, D] f64 into the slots `slot` of the pages `ids`."""
    n, n_kv, page = pages.shape[:3]
    hd = x.shape[-1]
    codes, step, base = _quantise(x)
    words = (codes.view(*codes.shape[:-1], -1, 8) << torch.tensor(SHIFTS, device=DEV, dtype=I32)).sum(-1, dtype=I32)
    flat = pages.view(n, n_kv, -1)
    w = torch.arange(hd // 8, device=DEV)
    s = slot.long()[:, None]
    place = (s // 4 * (hd // 8) + w) * 4 + s % 4 if values else s * (hd // 8) + w  # [tokens, D / 8]
    kv = torch.arange(n_kv, device=DEV)[:, None]
    flat.view(I32)[ids.long()[:, None, None], kv, place[:, None]] = words
    place = page * hd // 8 + torch.arange(hd // 32, device=DEV) * page + s
    flat.view(I32)[ids.long()[:, None, None], kv, place[:, None]] = torch.stack([step, base], -1).view(I32)[..., 0]


# ---------------------------------------------------------------- the plain forms: append and attention

def _rotate(x, cos, sin, interleaved):
    """x [.., heads, D] by cos, sin [.., rot / 2]: the first rot dimensions turned in pairs."""
    h = cos.shape[-1]
    c, s = cos[..., None, :], sin[..., None, :]
    if interleaved:
        a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., :h], x[..., h:2 * h]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, x[..., 2 * h:]], -1)


def _token_rows(s):
    """Each token's sequence, its place among the sequence's new tokens, and its position."""
    t = torch.arange(s["tokens"], device=DEV, dtype=I32)
    seq = torch.searchsorted(s["q_start"][1:].contiguous(), t, right=True)
    i = t - s["q_start"][seq]
    n = s["q_start"][seq + 1] - s["q_start"][seq]
    return seq, i, s["context"][seq] - n + i


def _plain_append(s, case):
    """In 64 bits: values next to the border of two codes."""
    heads, n_kv, hd = case["heads"], case["n_kv"], case["head_dim"]
    seq, _, pos = _token_rows(s)
    x = s["qkv"].double().view(s["tokens"], heads + 2 * n_kv, hd)
    q, k, v = x[:, :heads], x[:, heads:heads + n_kv], x[:, heads + n_kv:]
    if s["norms"] is not None:
        q = q / (q.square().mean(-1, keepdim=True) + 1e-6).sqrt() * s["norms"][0]
        k = k / (k.square().mean(-1, keepdim=True) + 1e-6).sqrt() * s["norms"][1]
    p = pos.long()
    c, sn = s["cos"][p].double(), s["sin"][p].double()
    ids, slot = s["pages"][seq, p // case["page"]], p % case["page"]
    _write(s["k"], False, _rotate(k, c, sn, case["interleaved"]), ids, slot)
    _write(s["v"], True, v, ids, slot)
    return _rotate(q, c, sn, case["interleaved"]).half(), _unpack(s["k"], False), _unpack(s["v"], True)


def _plain_attention(s, case):
    b, hd, n_kv, g = case["b"], case["head_dim"], case["n_kv"], case["heads"] // case["n_kv"]
    q_len = s["q_start"][1:] - s["q_start"][:-1]
    i = torch.arange(case["q"], device=DEV)
    q = s["q"].float()[(s["q_start"][:-1, None] + i).clamp(max=s["tokens"] - 1).long()]  # [b, q, heads, D], padded
    q = q.view(b, case["q"], n_kv, g, hd).permute(0, 2, 3, 1, 4).reshape(b, n_kv, g * case["q"], hd)
    k, v = s["k"], s["v"]
    if case["bits"] == 4:
        k, v = _unpack(k, False), _unpack(v, True)
    of = lambda t: t[s["pages"].clamp(min=0).long()].permute(0, 2, 1, 3, 4).reshape(b, n_kv, -1, hd).float()  # noqa: E731
    k, v = of(k), of(v)
    pos = (s["context"] - q_len)[:, None] + i  # [b, q]
    j = torch.arange(k.shape[2], device=DEV)
    seen = j <= pos[..., None]
    if case["window"]:
        seen &= (j > pos[..., None] - case["window"]) | (j < case["sinks"])
    a = torch.matmul(q * hd ** -0.5, k.transpose(-1, -2)).view(b, n_kv, g, case["q"], -1)
    a = a.masked_fill(~seen[:, None, None], -math.inf)
    a = (a - a.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    o = torch.matmul(a.view(b, n_kv, g * case["q"], -1), v).view(b, n_kv, g, case["q"], hd)
    o = o / a.sum(-1, keepdim=True).clamp(min=1e-30)
    seq, at, _ = _token_rows(s)
    return o.permute(0, 3, 1, 2, 4).reshape(b, case["q"], case["heads"], hd)[seq, at.long()].half()


# ---------------------------------------------------------------- the plain forms: pages

def _held(table, n):
    """Which entries hold a page, and the pages (0 for the others)."""
    held = (table >= 0) & (table < n)
    return held, table.masked_fill(~held, 0).long()


def _count(refs, ids, which, by):
    refs.index_add_(0, ids[which], torch.full((), by, dtype=I32, device=DEV).expand(int(which.sum())))


def _plain_fork(table, refs, parent):
    """Rows take their parents' entries (none: -1); counts follow the entries."""
    has = (parent >= 0) & (parent < table.shape[0])
    new = torch.where(has[:, None], table[parent.masked_fill(~has, 0).long()], -1)
    held, ids = _held(new, refs.numel())
    _count(refs, ids, held, 1)
    held, ids = _held(table, refs.numel())
    _count(refs, ids, held, -1)
    return new


def _plain_claim(table, refs, q_start, context, page):
    """Pages of their own for the positions that each sequence is about to write, the lowest free ones in order of sequence and
    block; (src, dst) of what has to be copied, and how many pages lack (then nothing changes)."""
    b, m = table.shape
    n, c = (q_start[1:] - q_start[:-1]).clamp(min=0), context
    j = torch.arange(m, device=DEV)
    at = (c - n).clamp(min=0)
    writes = (j >= (at // page)[:, None]) & (j * page < c[:, None]) & (n > 0)[:, None]
    held, ids = _held(table, refs.numel())
    owners = refs[ids].masked_fill(~held, 0)
    shared = writes & (owners > 1)
    # of the c that write to a page of r owners the first r - 1 copy it: their rank in order
    flat = shared.flatten().nonzero()[:, 0]
    of = ids.flatten()[flat]
    order = of.sort(stable=True).indices
    sorted_of = of[order]
    rank = torch.empty_like(of)
    rank[order] = torch.arange(of.numel(), device=DEV) - torch.searchsorted(sorted_of, sorted_of)
    copies = torch.zeros(b * m, dtype=torch.bool, device=DEV)
    copies[flat] = rank < owners.flatten()[flat] - 1
    copies = copies.view(b, m)
    need = (writes & (owners < 1)) | copies
    free = (refs < 1).nonzero()[:, 0].to(I32)
    lacking = (need.sum() - free.numel()).clamp(min=0).to(I32).view(1)
    none = torch.full((b,), -1, dtype=I32, device=DEV)
    if int(lacking) > 0:
        return none, none.clone(), lacking
    got = free[:int(need.sum())]
    first = copies & (j == (at // page)[:, None]) & (at % page > 0)[:, None]
    src = torch.where(first, table, -1).amax(1)
    _count(refs, ids, copies, -1)
    refs[got.long()] = 1
    table[need] = got
    return src, torch.where(first, table, -1).amax(1), lacking


def _plain_trim(table, refs, context, page, window, sinks):
    """Entries of positions that no later token sees become -1."""
    j = torch.arange(table.shape[1], device=DEV) * page
    gone = (j >= sinks) & (j + page <= (context - window + 1)[:, None])
    held, ids = _held(table, refs.numel())
    _count(refs, ids, held & gone, -1)
    table[gone] = -1


def _plain_compact(table, refs):
    """Used pages past the count of them move to the free places below it, in order."""
    used, n = refs > 0, refs.numel()
    count = used.sum().to(I32).view(1)
    u = int(count)
    movers, holes = used[u:].nonzero()[:, 0] + u, (~used[:u]).nonzero()[:, 0]
    moved = torch.where(used, torch.arange(n, device=DEV), -1).to(I32)
    moved[movers] = holes.to(I32)
    held, ids = _held(table, n)
    table.copy_(torch.where(held, moved[ids], -1))
    refs[holes] = refs[movers]
    refs[u:] = 0
    src, dst = torch.full((2, n), -1, dtype=I32, device=DEV)
    src[:movers.numel()], dst[:holes.numel()] = movers.to(I32), holes.to(I32)
    return src, dst, count


def _plain_copy(caches, src, dst):
    n = caches[0].shape[0]
    pairs = (src >= 0) & (src < n) & (dst >= 0) & (dst < n)
    a, b = src[pairs].long(), dst[pairs].long()
    for t in caches:
        t[b] = t[a]


def _plain_pages(s, case):
    k, v, refs = s["k"], s["v"], s["refs"].clone()
    if case["kind"] == "fork":
        table = _plain_fork(s["pages"], refs, s["parent"])
        src, dst, count = _plain_claim(table, refs, s["q_start"], s["context"], case["page"])
    else:
        table = s["pages"].clone()
        _plain_trim(table, refs, s["context"], case["page"], case["window"], case["sinks"])
        src, dst, count = _plain_compact(table, refs)
    _plain_copy([k, v], src, dst)
    return table, refs, src, dst, count, k, v


PLAIN = {"append": _plain_append, "attention": _plain_attention, "fork": _plain_pages, "compact": _plain_pages}


def _own(s, case):
    if os.path.join(os.getcwd(), "dream-tts_amd") not in sys.path:
        sys.path.insert(0, os.path.join(os.getcwd(), "dream-tts_amd"))
    from dtts import serving

    if case["kind"] == "append":
        q = serving.qk_rope_append_paged(s["qkv"], s["cos"], s["sin"], s["k"], s["v"], s["q_start"], s["context"], s["pages"],
                                         case["heads"], norms=s["norms"], eps=1e-6, interleaved=case["interleaved"])
        return q, *serving.unpack_pages(s["k"], s["v"])
    if case["kind"] == "attention":
        return serving.paged_attention(s["q"], s["k"], s["v"], s["q_start"], s["context"], s["pages"], max_q=case["q"],
                                       max_context=case["ctx"], scale=case["head_dim"] ** -0.5, window=case["window"],
                                       sinks=case["sinks"])
    refs = s["refs"].clone()
    if case["kind"] == "fork":
        table = serving.fork_pages(s["pages"], refs, s["parent"])
        src, dst, count = serving.claim_pages(table, refs, s["q_start"], s["context"], case["page"])
    else:
        table = s["pages"].clone()
        serving.trim_pages(table, refs, s["context"], case["page"], case["window"], sinks=case["sinks"])
        src, dst, count = serving.compact_pages(table, refs)
    serving.copy_pages([s["k"], s["v"]], src, dst)
    return table, refs, src, dst, count, s["k"], s["v"]


def run(state):
    case = state["case"]
    return _own(state, case) if own else PLAIN[case["kind"]](state, case)


# ---------------------------------------------------------------- what a pass cannot do without

def _page_bytes(case):
    """Of one page's keys, or values."""
    return case["n_kv"] * case["page"] * (2 * case["head_dim"] if case["bits"] == 16 else 5 * case["head_dim"] // 8)


def _used(case):
    """Of a fragmented pool: the entries of its table, and how many pages move."""
    rng = random.Random(case["lens"])
    page, longest = case["page"], -(-case["ctx"] // case["page"])
    ids = np.random.RandomState(case["lens"]).permutation(case["pool"])
    used, at = np.zeros(case["pool"], bool), 0
    for s in range(case["b"]):
        c = case["ctx"] if s == 0 else rng.randint(1, case["ctx"])
        k = -(-c // page)
        if s % 3 != 2:
            j = np.arange(k) * page
            used[ids[at:at + k][(j < case["sinks"]) | (j + page > c - case["window"] + 1)]] = True
        at += k
    return case["b"] * longest, int(used[int(used.sum()):].sum())


def work(case):
    kind = case["kind"]
    if kind == "compact":
        entries, moves = _used(case)
        return dict(bytes=4 * (2 * case["pool"] + 2 * entries + 2 * case["pool"]) + 4 * moves * _page_bytes(case), flops=entries)
    if kind == "fork":
        b = case["groups"] * case["beams"]
        entries = b * (-(-case["ctx"] // case["page"]) + 2)
        # of a row in seven that ends, and of each request's beams one keeps its page
        copies = max(0, int(b * 6 / 7) - case["groups"])
        return dict(bytes=4 * (2 * entries + 2 * case["pool"] + 7 * b) + 4 * copies * _page_bytes(case), flops=entries)
    n, c = _lengths(case)
    hd, heads, n_kv = case["head_dim"], case["heads"], case["n_kv"]
    if kind == "append":
        e, pages = 2 if case["dtype"] == "f16" else 4, sum(-(-x // case["page"]) for x in c) + 3
        read = 2 * pages * case["page"] * n_kv * (5 * hd // 8 + 2 * hd)  # the values that the pages stand for
        return dict(bytes=sum(n) * ((heads + 2 * n_kv) * hd * e + heads * hd * 2 + 2 * n_kv * 5 * hd // 8 + 4 * case["rot"]) + read,
                    flops=6 * sum(n) * heads * hd + 4 * pages * case["page"] * n_kv * hd)
    window, row = case["window"] or max(c), 5 * hd // 8 if case["bits"] == 4 else 2 * hd

    def seen(p):
        return min(p + 1, window) + min(case["sinks"], max(0, p + 1 - window))

    pairs = sum(seen(p) for k, x in zip(n, c) for p in range(x - k, x))
    rows = sum(min(x, window + k - 1 + case["sinks"]) for k, x in zip(n, c) if k)
    return dict(bytes=2 * 2 * sum(n) * heads * hd + 2 * rows * n_kv * row, flops=4 * hd * heads * pairs)


# ---------------------------------------------------------------- the definitions in 64 bits

def _host(t):
    return t.cpu().double().numpy()


def _row_values(pages, hd, values):
    """What 4-bit pages stand for, [n, n_kv, page, D] f64, from their bytes on the host."""
    raw = pages.cpu().numpy()
    n, n_kv, page = raw.shape[:3]
    raw = raw.reshape(n, n_kv, -1)
    bits = np.ascontiguousarray(raw[..., :page * hd // 2]).view("<u4")
    bits = bits.reshape(n, n_kv, page // 4, hd // 8, 4).swapaxes(-1, -2) if values else bits
    bits = bits.reshape(n, n_kv, page, hd // 8)
    out = np.empty((n, n_kv, page, hd // 8, 8))
    for e in range(8):
        out[..., e] = 64 + (bits >> (4 * (e // 2) + 16 * (e % 2)) & 15)
    pairs = np.ascontiguousarray(raw[..., page * hd // 2:]).view("<f2").astype(np.float64).reshape(n, n_kv, hd // 32, page, 2)
    pairs = pairs.transpose(0, 1, 3, 2, 4)[..., None, :]
    x = out.reshape(n, n_kv, page, hd // 32, 32) * pairs[..., 0] + pairs[..., 1]
    return x.astype(np.float16).astype(np.float64).reshape(n, n_kv, page, hd)


def _group_values(x):
    """What rows [.., D] f64 become in 4 bits."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    lo = g.min(-1, keepdims=True)
    d = ((g.max(-1, keepdims=True) - lo) / 15).astype(np.float16).astype(np.float64)
    b = (lo - 64 * d).astype(np.float16).astype(np.float64)
    c = np.where(d > 0, np.clip(np.rint((g - b) / np.where(d > 0, d, 1.0)), 64, 79), 64)
    return (c * d + b).astype(np.float16).astype(np.float64).reshape(x.shape)


def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return None
    s = prepare(case, seed)
    start, ctx = s["q_start"].tolist(), s["context"].tolist()
    n_kv, hd, page, heads = case["n_kv"], case["head_dim"], case["page"], case["heads"]
    if case["kind"] == "append":
        pos = np.concatenate([np.arange(c - (e - a), c) for a, e, c in zip(start, start[1:], ctx)])
        x = _host(s["qkv"]).reshape(s["tokens"], heads + 2 * n_kv, hd)
        if case["norm"]:
            g = _host(s["norms"])
            x[:, :heads] = x[:, :heads] / np.sqrt(np.mean(x[:, :heads] ** 2, -1, keepdims=True) + 1e-6) * g[0]
            k = x[:, heads:heads + n_kv]
            x[:, heads:heads + n_kv] = k / np.sqrt(np.mean(k ** 2, -1, keepdims=True) + 1e-6) * g[1]
        turn = _host(s["cos"])[pos] + 1j * _host(s["sin"])[pos]
        h, y = case["rot"] // 2, x[:, :heads + n_kv].copy()
        one, two = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if case["interleaved"] else (slice(0, h), slice(h, 2 * h))
        z = (y[..., one] + 1j * y[..., two]) * turn[:, None]
        y[..., one], y[..., two] = z.real, z.imag
        k, v, table = _row_values(s["k"], hd, False), _row_values(s["v"], hd, True), s["pages"].cpu().numpy()
        kn, vn = _group_values(y[:, heads:]), _group_values(x[:, heads + n_kv:])
        for i, (a, e) in enumerate(zip(start, start[1:])):
            for t in range(a, e):
                at = table[i, pos[t] // page], slice(None), pos[t] % page
                k[at], v[at] = kn[t], vn[t]
        return y[:, :heads], k, v
    out = torch.zeros(s["q"].shape, dtype=F64, device=DEV)
    g = heads // n_kv
    k, v = s["k"], s["v"]
    if case["bits"] == 4:
        k, v = (torch.from_numpy(_row_values(t, hd, i)).half().to(DEV) for t, i in ((k, False), (v, True)))  # f16 already
    for i, (a, e, c) in enumerate(zip(start, start[1:], ctx)):
        if e == a:
            continue
        first = c - (e - a)
        lo = max(0, first - case["window"] + 1) if case["window"] else 0  # the keys that some row sees
        j = torch.cat([torch.arange(min(case["sinks"], lo), device=DEV), torch.arange(lo, c, device=DEV)])
        at = s["pages"][i].long()[j // page], slice(None), j % page
        ks, vs = k[at].double(), v[at].double()  # [keys, n_kv, D]
        pos = torch.arange(first, c, device=DEV)[:, None]
        hidden = j > pos
        if case["window"]:
            hidden |= (j <= pos - case["window"]) & (j >= case["sinks"])
        for h in range(heads):
            z = s["q"][a:e, h].double() @ ks[:, h // g].T.contiguous() / math.sqrt(hd)
            out[a:e, h] = z.masked_fill(hidden, -math.inf).softmax(-1) @ vs[:, h // g].contiguous()
    return out
