"""The operators of a serving step, as measurable cases.

A case is a dict of plain values; ``kind`` says which operator it goes through:

  rotary     rotary positions on [rows, heads, D] (``dtts.serving.rotary``)
  append     QK-norm, rotary positions and the write into a paged cache
             (``dtts.serving.qk_rope_append_paged``)
  attention  attention of each sequence's new tokens over its pages
             (``dtts.serving.paged_attention``)
  sample     tokens from logits and given random numbers (``dtts.serving.sample``)

Lengths of ragged batches follow from the case alone; values follow from the seed.
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
        # a long document's prompt (many rows, far positions on a table scaled for them) before a
        # cache of the caller's own
        dict(name="rotary_f16_8192", kind="rotary", dtype="f16", rows=8192, heads=32, head_dim=128, rot=128,
             interleaved=False, length=131072, scaling="yarn", factor=8.0),
        # an odd number of f32 rows, a quarter of the head rotated in interleaved pairs
        dict(name="rotary_f32_777_part", kind="rotary", dtype="f32", rows=777, heads=16, head_dim=64, rot=16,
             interleaved=True, length=4096, scaling="linear", factor=4.0),
        # a talker's decode step: one f32 row of q, k and v per lane, with QK-norm
        dict(name="append_decode_48", kind="append", dtype="f32", b=48, prefills=0, q=1, ctx=1536, heads=16, n_kv=8,
             head_dim=128, rot=128, interleaved=False, norm=True, page=16, lens=1),
        # prompts of several requests at once, f16 rows, half of a 64-wide head rotated
        dict(name="append_prefill_7", kind="append", dtype="f16", b=7, prefills=7, q=1301, ctx=4000, heads=32, n_kv=8,
             head_dim=64, rot=32, interleaved=True, norm=False, page=64, lens=2),
        # one request, one token, a short context: the smallest call
        dict(name="attention_1x1_300", kind="attention", b=1, prefills=0, q=1, ctx=300, heads=16, n_kv=8, head_dim=128,
             page=16, window=0, lens=3),
        # a talker's batch, every lane at its own position
        dict(name="attention_48x1_1536", kind="attention", b=48, prefills=0, q=1, ctx=1536, heads=16, n_kv=8,
             head_dim=128, page=16, window=0, lens=4),
        # few requests with very long contexts, eight query heads a kv head
        dict(name="attention_5x1_65000", kind="attention", b=5, prefills=0, q=1, ctx=65000, heads=32, n_kv=4,
             head_dim=128, page=64, window=0, lens=5),
        # a long prompt's chunk after what is already cached
        dict(name="attention_1x2048_10000", kind="attention", b=1, prefills=1, q=2048, ctx=10000, heads=32, n_kv=8,
             head_dim=128, page=64, window=0, lens=6),
        # a mixed batch: two prompts' chunks beside 30 decoding requests, 64-wide heads, a sliding window
        dict(name="attention_mixed_32", kind="attention", b=32, prefills=2, q=501, ctx=3001, heads=16, n_kv=4,
             head_dim=64, page=32, window=1024, lens=7),
        # a code predictor's codebook for a talker's batch
        dict(name="sample_48x2048", kind="sample", dtype="f32", rows=48, vocab=2048, lens=8),
        # a text vocabulary for a large batch
        dict(name="sample_64x131072", kind="sample", dtype="f32", rows=64, vocab=131072, lens=9),
        # few rows of an odd vocabulary in f16, where many logits are equal
        dict(name="sample_3x50021_f16", kind="sample", dtype="f16", rows=3, vocab=50021, lens=10),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "attention", "attention", "attention", "sample", "sample"])
    if kind == "rotary":
        hd = rng.choice([64, 128])
        return dict(kind=kind, dtype=rng.choice(["f16", "f32"]), rows=_log_int(rng, 1, 4096), heads=rng.choice([1, 8, 16, 32]),
                    head_dim=hd, rot=rng.choice([hd, hd, hd // 2, hd // 4]), interleaved=rng.random() < 0.5,
                    length=_log_int(rng, 2048, 131072), scaling=rng.choice(["none", "linear", "ntk", "yarn"]), factor=4.0)
    if kind == "sample":
        vocab = _log_int(rng, 100, 160000)
        return dict(kind=kind, dtype=rng.choice(["f32", "f32", "f16"]), rows=_log_int(rng, 1, min(256, 8000000 // vocab)),
                    vocab=vocab, lens=rng.randrange(1 << 20))
    hd = rng.choice([64, 128, 128])
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
        return dict(case, dtype=rng.choice(["f32", "f16"]), ctx=q + _log_int(rng, 1, 8000), norm=rng.random() < 0.5,
                    rot=rng.choice([hd, hd, hd // 2]), interleaved=rng.random() < 0.3)
    most = min(66000, int(6e8) // (b * q * heads), int(4e9) // (b * n_kv * hd * 8))
    return dict(case, ctx=q + _log_int(rng, 1, max(2, most - q)), window=rng.choice([0, 0, 0, _log_int(rng, 16, 4096)]))


# ---------------------------------------------------------------- inputs from the seed alone

class _Draw:
    """torch's generator on the device, one stream per seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def normal(self, shape, std=1.0):
        return torch.randn(shape, generator=self.g, device=DEV) * std

    def uniform(self, n, lo, hi):
        return torch.rand(n, generator=self.g, device=DEV) * (hi - lo) + lo

    def ints(self, shape, lo, hi):
        return torch.randint(lo, hi, shape, generator=self.g, device=DEV)


def _dtype(case):
    return F16 if case["dtype"] == "f16" else F32


def _inv_freq(rot, base, scaling, factor, original):
    """Angles per position [rot / 2], f64, and the factor on cos and sin, of a table for `factor` times
    the trained length: positions divided (linear), the base raised (ntk), or by wavelength (yarn)."""
    i = np.arange(0, rot, 2, dtype=np.float64) / rot
    if scaling == "linear":
        return base ** -i / factor, 1.0
    if scaling == "ntk":
        return (base * factor ** (rot / max(rot - 2, 1))) ** -i, 1.0
    if scaling == "yarn":
        def at(turns):
            return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = np.clip((np.arange(rot // 2) - low) / max(high - low, 1e-3), 0, 1)
        return base ** -i / factor * ramp + base ** -i * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return base ** -i, 1.0


def _tables(length, rot, scaling="none", factor=1.0):
    f, m = _inv_freq(rot, 1e6, scaling, factor, length / factor)
    a = torch.arange(length, device=DEV, dtype=F64)[:, None] * torch.from_numpy(f).to(DEV)[None]
    return (a.cos() * m).float(), (a.sin() * m).float()


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


def _batch(case, seed):
    """q_start, contexts and the page table of a ragged batch: its pages scattered over a pool, -1 past a
    sequence's last."""
    n, c = _lengths(case)
    page = case["page"]
    counts = [-(-x // page) for x in c]
    pool = sum(counts) + 3
    rng = np.random.RandomState(seed % (1 << 31))
    order = rng.permutation(pool)
    table = np.full((case["b"], max(counts)), -1, np.int32)
    at = 0
    for i, k in enumerate(counts):
        table[i, :k] = order[at:at + k]
        at += k
    start = np.concatenate([[0], np.cumsum(n)])
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)  # noqa: E731
    return dict(q_start=dev(start), context=dev(c), pages=dev(table), tokens=int(start[-1]), pool=pool)


def prepare(case, seed):
    d, kind = _Draw(seed), case["kind"]
    if kind == "rotary":
        cos, sin = _tables(case["length"], case["rot"], case["scaling"], case["factor"])
        x = d.normal((case["rows"], case["heads"], case["head_dim"])).to(_dtype(case))
        return dict(case=case, x=x, cos=cos, sin=sin, pos=d.ints((case["rows"],), 0, case["length"]).to(I32))
    if kind == "sample":
        rows, vocab, rng = case["rows"], case["vocab"], random.Random(case["lens"])
        logits = d.normal((rows, vocab), 2.5)
        # a few likely tokens over the rest, and the tokens that a server suppresses
        logits.scatter_add_(1, d.ints((rows, 12), 0, vocab), d.uniform((rows, 12), 4.0, 10.0))
        logits[:, vocab - vocab // 50:] = -math.inf
        # requests' own settings: greedy ones, plain temperature, each filter alone, all of them
        style = [rng.randrange(7) for _ in range(rows)]
        col = lambda off, on, which, t: torch.tensor([on() if s in which else off for s in style], dtype=t, device=DEV)  # noqa: E731
        return dict(case=case, logits=logits.to(_dtype(case)), u=d.uniform((rows,), 0.0, 1.0).clamp_(max=1 - 2.0 ** -24),
                    temperature=col(0.0, lambda: rng.uniform(0.6, 1.2), (1, 2, 3, 4, 5, 6), F32),
                    top_k=col(0, lambda: min(vocab, rng.choice([1, 20, 50, 400])), (2, 5, 6), I32),
                    top_p=col(1.0, lambda: rng.uniform(0.5, 0.99), (3, 5, 6), F32),
                    min_p=col(0.0, lambda: rng.uniform(0.01, 0.1), (4, 6), F32))
    s = dict(case=case, **_batch(case, seed))
    shape = (s["pool"], case["n_kv"], case["page"], case["head_dim"])
    s["k"], s["v"] = d.normal(shape, 1.3).half(), d.normal(shape).half()
    if kind == "attention":
        s["q"] = d.normal((s["tokens"], case["heads"], case["head_dim"]), 1.3).half()
        return s
    s["qkv"] = d.normal((s["tokens"], (case["heads"] + 2 * case["n_kv"]) * case["head_dim"])).to(_dtype(case))
    s["cos"], s["sin"] = _tables(case["ctx"], case["rot"])
    s["norms"] = d.uniform((2, case["head_dim"]), 0.8, 1.2) if case["norm"] else None
    return s


# ---------------------------------------------------------------- the plain forms

def _rotate(x, cos, sin, interleaved):
    """x [.., heads, D] f32 by cos, sin [.., rot / 2]: the first rot dimensions turned in pairs."""
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


def _plain_rotary(s, case):
    p = s["pos"].long()
    return _rotate(s["x"].float(), s["cos"][p], s["sin"][p], case["interleaved"]).to(s["x"].dtype)


def _plain_append(s, case):
    heads, n_kv, hd = case["heads"], case["n_kv"], case["head_dim"]
    seq, _, pos = _token_rows(s)
    x = s["qkv"].float().view(s["tokens"], heads + 2 * n_kv, hd)
    q, k, v = x[:, :heads], x[:, heads:heads + n_kv], x[:, heads + n_kv:]
    if s["norms"] is not None:
        q = q / (q.square().mean(-1, keepdim=True) + 1e-6).sqrt() * s["norms"][0]
        k = k / (k.square().mean(-1, keepdim=True) + 1e-6).sqrt() * s["norms"][1]
    p = pos.long()
    q = _rotate(q, s["cos"][p], s["sin"][p], case["interleaved"]).half()
    k = _rotate(k, s["cos"][p], s["sin"][p], case["interleaved"]).half()
    at = s["pages"][seq, p // case["page"]].long(), slice(None), p % case["page"]
    s["k"][at], s["v"][at] = k, v.half()
    return q, s["k"], s["v"]


def _plain_attention(s, case):
    b, hd, n_kv, g = case["b"], case["head_dim"], case["n_kv"], case["heads"] // case["n_kv"]
    q_len = s["q_start"][1:] - s["q_start"][:-1]
    i = torch.arange(case["q"], device=DEV)
    q = s["q"].float()[(s["q_start"][:-1, None] + i).clamp(max=s["tokens"] - 1).long()]  # [b, q, heads, D], padded
    q = q.view(b, case["q"], n_kv, g, hd).permute(0, 2, 3, 1, 4).reshape(b, n_kv, g * case["q"], hd)
    of = lambda t: t[s["pages"].clamp(min=0).long()].permute(0, 2, 1, 3, 4).reshape(b, n_kv, -1, hd).float()  # noqa: E731
    k, v = of(s["k"]), of(s["v"])
    pos = (s["context"] - q_len)[:, None] + i  # [b, q]
    j = torch.arange(k.shape[2], device=DEV)
    seen = j <= pos[..., None]
    if case["window"]:
        seen &= j > pos[..., None] - case["window"]
    a = torch.matmul(q * hd ** -0.5, k.transpose(-1, -2)).view(b, n_kv, g, case["q"], -1)
    a = a.masked_fill(~seen[:, None, None], -math.inf)
    a = (a - a.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    o = torch.matmul(a.view(b, n_kv, g * case["q"], -1), v).view(b, n_kv, g, case["q"], hd)
    o = o / a.sum(-1, keepdim=True).clamp(min=1e-30)
    seq, at, _ = _token_rows(s)
    return o.permute(0, 3, 1, 2, 4).reshape(b, case["q"], case["heads"], hd)[seq, at.long()].half()


def _plain_sample(s, case):
    """In 64 bits: sums over a vocabulary decide which token a random number falls on."""
    x = s["logits"].double()
    x = x.masked_fill(x.isnan(), -math.inf)
    top = x.amax(1, keepdim=True)
    greedy = ~(s["temperature"] > 0)
    w = ((x - top) / s["temperature"].masked_fill(greedy, 1.0).double()[:, None]).exp().masked_fill(x == top, 1.0)
    order = x.sort(dim=1, descending=True, stable=True).indices  # equal logits: the lower index first
    rank = torch.arange(x.shape[1], device=DEV)
    k = s["top_k"].masked_fill(s["top_k"] <= 0, x.shape[1])[:, None]
    ws = w.gather(1, order).masked_fill(rank >= k, 0.0)
    c = ws.cumsum(1)
    before = torch.cat([torch.zeros_like(c[:, :1]), c[:, :-1]], 1)
    p, m = s["top_p"].double()[:, None], s["min_p"].double()[:, None]
    keep = (rank < k) & ((before < p * c[:, -1:]) | (p >= 1)) & (ws >= m) | (rank == 0)
    kept = torch.zeros_like(keep).scatter(1, order, keep)
    wk = w.masked_fill(~kept, 0.0).cumsum(1)
    token = torch.searchsorted(wk, s["u"].double()[:, None] * wk[:, -1:], right=True)
    token = torch.where(greedy[:, None], order[:, :1], token)
    logprob = (w.gather(1, token) / wk[:, -1:]).log().masked_fill(greedy[:, None], 0.0)
    return token[:, 0].to(I32), logprob[:, 0].float()


PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}


def _own(s, case):
    if os.path.join(os.getcwd(), "dream-tts_amd") not in sys.path:
        sys.path.insert(0, os.path.join(os.getcwd(), "dream-tts_amd"))
    from dtts import serving

    if case["kind"] == "rotary":
        return serving.rotary(s["x"], s["cos"], s["sin"], s["pos"], interleaved=case["interleaved"])
    if case["kind"] == "append":
        q = serving.qk_rope_append_paged(s["qkv"], s["cos"], s["sin"], s["k"], s["v"], s["q_start"], s["context"], s["pages"],
                                         case["heads"], norms=s["norms"], eps=1e-6, interleaved=case["interleaved"])
        return q, s["k"], s["v"]
    if case["kind"] == "attention":
        return serving.paged_attention(s["q"], s["k"], s["v"], s["q_start"], s["context"], s["pages"], max_q=case["q"],
                                       max_context=case["ctx"], scale=case["head_dim"] ** -0.5, window=case["window"])
    return serving.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                          min_p=s["min_p"])


def run(state):
    case = state["case"]
    return _own(state, case) if own else PLAIN[case["kind"]](state, case)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * (2 if case["dtype"] == "f16" else 4) + 28 * case["rows"], flops=4 * n)
    if kind == "rotary":
        n, e = case["rows"] * case["heads"] * case["head_dim"], 2 if case["dtype"] == "f16" else 4
        return dict(bytes=2 * e * n + case["rows"] * (4 + 4 * case["rot"]), flops=3 * n)
    n, c = _lengths(case)
    hd, heads, n_kv = case["head_dim"], case["heads"], case["n_kv"]
    if kind == "append":
        e = 2 if case["dtype"] == "f16" else 4
        return dict(bytes=sum(n) * ((heads + 2 * n_kv) * hd * (e + 2) + 4 * case["rot"]), flops=6 * sum(n) * heads * hd)
    window = case["window"] or max(c)
    pairs = sum(min(p + 1, window) for k, x in zip(n, c) for p in range(x - k, x))
    rows = sum(min(x, window + k - 1) for k, x in zip(n, c) if k)
    return dict(bytes=2 * (2 * sum(n) * heads * hd + 2 * rows * n_kv * hd), flops=4 * hd * heads * pairs)


# ---------------------------------------------------------------- the definitions in 64 bits

def _turned(x, angle_cos, angle_sin, interleaved):
    """numpy f64 [n, heads, D] times the rotation e^{i angle}, as complex numbers."""
    h = angle_cos.shape[1]
    z = x[..., 0:2 * h:2] + 1j * x[..., 1:2 * h:2] if interleaved else x[..., :h] + 1j * x[..., h:2 * h]
    z = z * (angle_cos + 1j * angle_sin)[:, None]
    y = x.copy()
    if interleaved:
        y[..., 0:2 * h:2], y[..., 1:2 * h:2] = z.real, z.imag
    else:
        y[..., :h], y[..., h:2 * h] = z.real, z.imag
    return y


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    host = lambda t: t.cpu().double().numpy()  # noqa: E731
    if kind == "rotary":
        p = s["pos"].long()
        return _turned(host(s["x"]), host(s["cos"][p]), host(s["sin"][p]), case["interleaved"])
    if kind == "sample":
        return _exact_sample(s, case)
    start, ctx = s["q_start"].tolist(), s["context"].tolist()
    n_kv, hd, page = case["n_kv"], case["head_dim"], case["page"]
    if kind == "append":
        heads = case["heads"]
        pos = np.concatenate([np.arange(c - (e - a), c) for a, e, c in zip(start, start[1:], ctx)])
        x = host(s["qkv"]).reshape(s["tokens"], heads + 2 * n_kv, hd)
        if case["norm"]:
            g = host(s["norms"])
            x[:, :heads] = x[:, :heads] / np.sqrt(np.mean(x[:, :heads] ** 2, -1, keepdims=True) + 1e-6) * g[0]
            k = x[:, heads:heads + n_kv]
            x[:, heads:heads + n_kv] = k / np.sqrt(np.mean(k ** 2, -1, keepdims=True) + 1e-6) * g[1]
        turned = _turned(x[:, :heads + n_kv], host(s["cos"])[pos], host(s["sin"])[pos], case["interleaved"])
        k, v, table = host(s["k"]), host(s["v"]), s["pages"].cpu().numpy()
        for i, (a, e) in enumerate(zip(start, start[1:])):
            for t in range(a, e):
                at = table[i, pos[t] // page], slice(None), pos[t] % page
                k[at], v[at] = turned[t, heads:], x[t, heads + n_kv:]
        return turned[:, :heads], k, v
    out = torch.zeros(s["q"].shape, dtype=F64, device=DEV)
    g = case["heads"] // n_kv
    for i, (a, e, c) in enumerate(zip(start, start[1:], ctx)):
        if e == a:
            continue
        ids = s["pages"][i, :-(-c // page)].long()
        k, v = (t[ids].transpose(0, 1).reshape(n_kv, -1, hd)[:, :c].double() for t in (s["k"], s["v"]))
        j, pos = torch.arange(c, device=DEV), torch.arange(c - (e - a), c, device=DEV)[:, None]
        hidden = (j > pos) | (j <= pos - case["window"] if case["window"] else j < 0)
        for h in range(case["heads"]):
            z = s["q"][a:e, h].double() @ k[h // g].T.contiguous() / math.sqrt(hd)
            out[a:e, h] = z.masked_fill(hidden, -math.inf).softmax(-1) @ v[h // g]
    return out


def _exact_sample(s, case):
    """Row by row on the host: the tokens in their order of preference, cut where a filter says."""
    x, tokens, logprobs = host_rows(s["logits"]), [], []
    t, k, p, m, u = (s[a].cpu().double().numpy() for a in ("temperature", "top_k", "top_p", "min_p", "u"))
    for r in range(case["rows"]):
        order = np.argsort(-x[r], kind="stable")
        if not t[r] > 0:
            tokens.append(int(order[0]))
            logprobs.append(0.0)
            continue
        if 0 < k[r] < len(order):
            order = order[:int(k[r])]
        w = np.exp((x[r][order] - x[r][order[0]]) / t[r])
        most = len(order)
        if p[r] < 1:
            most = max(1, int(np.searchsorted(np.cumsum(w), p[r] * np.sum(w), side="left")) + 1)
        most = max(1, min(most, int(np.sum(w >= m[r]))))
        by_index = np.sort(order[:most])
        w = np.exp((x[r][by_index] - x[r][order[0]]) / t[r])
        c = np.cumsum(w)
        at = int(np.searchsorted(c, u[r] * c[-1], side="right"))
        tokens.append(int(by_index[at]))
        logprobs.append(math.log(w[at] / c[-1]))
    return np.array(tokens, np.int32), np.array(logprobs)


def host_rows(t):
    return t.cpu().double().numpy()
