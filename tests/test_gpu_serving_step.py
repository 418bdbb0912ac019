"""The serving ops as a server runs them: prompts, then single tokens of a batch that changes, through
projection, append, attention, projection and sampling; and the step captured in a graph."""
import numpy as np
import pytest
import torch

from dtts import ops, serving

import _serving_ref as ref

pytestmark = pytest.mark.gpu

HEADS, N_KV, HD, PAGE, DIM, VOCAB = 4, 2, 64, 16, 128, 500


class Model:
    """One attention layer between an embedding and a vocabulary, in the library's ops."""

    def __init__(self, dev, n_pages=64):
        g = torch.Generator().manual_seed(7)
        w = lambda *s: (torch.randn(s, generator=g) * 0.08).half().to(dev)  # noqa: E731
        self.embed, self.wqkv = w(VOCAB, DIM) * 12, w((HEADS + 2 * N_KV) * HD, DIM)
        self.wo, self.head = w(DIM, HEADS * HD), w(VOCAB - VOCAB % 16, DIM)
        self.norms = (torch.rand((2, HD), generator=g) + 0.5).to(dev)
        self.cos, self.sin = (torch.from_numpy(t).to(dev) for t in serving.rope_table_scaled(600, HD, 1e4, "yarn", 2.0, 300))
        # slots that hold nothing hold NaN
        self.k, self.v = (torch.full((n_pages, N_KV, PAGE, HD), float("nan"), dtype=torch.float16, device=dev) for _ in range(2))

    def step(self, x, start, ctx, pages, last, u, settings, max_q, max_context, ws=(None, None)):
        """x [tokens, DIM] f16 -> tokens and log-probabilities of the rows `last`."""
        qkv = ops.matmul_nt(x, self.wqkv)
        q = serving.qk_rope_append_paged(qkv, self.cos, self.sin, self.k, self.v, start, ctx, pages, HEADS, self.norms)
        o = serving.paged_attention(q, self.k, self.v, start, ctx, pages, max_q, max_context, HD ** -0.5, workspace=ws[0])
        h = ops.matmul_nt(o.view(x.shape[0], HEADS * HD), self.wo).half() + x
        logits = ops.matmul_nt(h[last], self.head)
        return serving.sample(logits, u, *settings, workspace=ws[1]), logits

    def whole(self, tokens):
        """The logits after a whole sequence, its attention in 64 bits, everything else as the steps have it."""
        x = self.embed[tokens]
        n = len(tokens)
        qkv = torch.cat([ops.matmul_nt(x[i:i + 64], self.wqkv) for i in range(0, n, 64)]).double().view(n, HEADS + 2 * N_KV, HD)
        w, pos = self.norms.double(), np.arange(n)
        qk = qkv[:, :HEADS + N_KV] / (qkv[:, :HEADS + N_KV].square().mean(-1, keepdim=True) + 1e-6).sqrt()
        qk = torch.cat([qk[:, :HEADS] * w[0], qk[:, HEADS:] * w[1]], 1).cpu().numpy()
        qk, _ = ref.turn(qk, self.cos.cpu().double().numpy()[pos], self.sin.cpu().double().numpy()[pos], False)
        qk = torch.from_numpy(qk).half().double()
        v = qkv[:, HEADS + N_KV:].half().double().cpu()
        o = torch.stack([torch.softmax(qk[:, HEADS + h // 2] @ qk[-1, h] * HD ** -0.5, 0) @ v[:, h // 2] for h in range(HEADS)])
        h = ops.matmul_nt(o.half().view(1, -1).to(x.device), self.wo).half() + x[-1:]
        return ops.matmul_nt(h, self.head)[0].double().cpu()


def _i32(a, dev):
    return torch.tensor(a, dtype=torch.int32, device=dev)


def test_a_server_of_changing_requests(dev):
    """Three requests with their own settings, one of them joining late and one leaving; pages handed out as
    contexts grow. Each step's logits match the whole sequence's, and its tokens the sampler's definition."""
    m = Model(dev)
    rng = np.random.RandomState(5)
    free = list(rng.permutation(64))
    prompts = [rng.randint(0, VOCAB, n).tolist() for n in (19, 1, 40)]
    setting = [(0.9, 50, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.2, 0, 0.8, 0.02)]
    seqs, tables, cached = [list(p) for p in prompts], [[] for _ in prompts], [0, 0, 0]
    for step in range(24):
        live = [i for i in range(3) if not (i == 2 and step < 4) and not (i == 1 and step >= 15)]
        n = [len(seqs[i]) - cached[i] for i in live]
        n[0] = min(n[0], 7)  # the first prompt goes in chunks
        ctx = [cached[i] + k for i, k in zip(live, n)]
        for i, c in zip(live, ctx):
            while len(tables[i]) * PAGE < c:
                tables[i].append(int(free.pop()))
        width = max(len(t) for t in tables) + 1
        pages = _i32([tables[i] + [-1] * (width - len(tables[i])) for i in live], dev)
        start = np.concatenate([[0], np.cumsum(n)])
        fed = sum((seqs[i][cached[i]:cached[i] + k] for i, k in zip(live, n)), [])
        u = rng.rand(len(live)).astype(np.float32)
        cols = [torch.tensor([setting[i][j] for i in live], dtype=torch.int32 if j == 1 else torch.float32, device=dev) for j in range(4)]
        (tok, lp), logits = m.step(m.embed[torch.tensor(fed, device=dev)], _i32(start, dev), _i32(ctx, dev), pages,
                                   torch.from_numpy(start[1:] - 1).to(dev), torch.from_numpy(u).to(dev), cols, max(n), max(ctx))
        for r, i in enumerate(live):
            cached[i] = ctx[r]
            want = m.whole(torch.tensor(seqs[i][:cached[i]], device=dev))
            # f16 steps of values up to 8 (2^-9 each) in q, k, v, the output and the residual, through a
            # projection of 128 terms of 0.08: 4 * 2^-9 * 0.08 * 128^(1/2) * 8 < 0.06
            assert float((logits[r].double().cpu() - want).abs().max()) < 0.06
            t, k, p, mp = setting[i]
            got = ref.sample(logits[r].cpu().double().numpy(), float(u[r]), float(np.float32(t)), k, float(np.float32(p)), float(np.float32(mp)))
            assert int(tok[r]) == got[0] and abs(float(lp[r]) - got[1]) < 1e-5
            if cached[i] == len(seqs[i]):
                seqs[i].append(int(tok[r]))
        if step == 15:
            free = tables[1] + free  # the finished request's pages, stale values and all, go to the others
            free = free[::-1]


def test_a_captured_step_is_replayed_while_lengths_change(dev):
    """One graph of append, attention and sampling for a padded batch: replays with other contexts, pages,
    settings and an idle slot, with eager work between them, each against the eager call."""
    b, cap = 6, 400
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn((b, (HEADS + 2 * N_KV) * HD), generator=g).to(dev)
    cos, sin = (torch.from_numpy(t).to(dev) for t in ops.rope_table_f32(512, HD, 1e4))
    pool = 200
    k, v = (torch.randn((pool, N_KV, PAGE, HD), generator=g).half().to(dev) for _ in range(2))
    head = (torch.randn((9008, HEADS * HD), generator=g) * 0.3).half().to(dev)
    start, ctx = _i32(list(range(b + 1)), dev), _i32([1] * b, dev)
    pages, u = _i32(np.full((b, cap // PAGE), -1), dev), torch.zeros(b, device=dev)
    temp, topk, topp = torch.ones(b, device=dev), _i32([0] * b, dev), torch.ones(b, device=dev)
    ws = torch.empty(max(serving.paged_attention_workspace_bytes(b, b, HEADS, N_KV, HD, 1, cap), 16), dtype=torch.uint8, device=dev)
    ws2 = torch.empty(max(serving.sample_workspace_bytes(b, 9008), 16), dtype=torch.uint8, device=dev)
    q, o = (torch.zeros((b, HEADS, HD), dtype=torch.float16, device=dev) for _ in range(2))
    gws = torch.empty(max(ops.gemm_workspace_bytes(b, HEADS * HD, 9008), 16), dtype=torch.uint8, device=dev)

    def step():
        serving.qk_rope_append_paged(qkv, cos, sin, k, v, start, ctx, pages, HEADS, out=q)
        serving.paged_attention(q, k, v, start, ctx, pages, 1, cap, HD ** -0.5, out=o, workspace=ws)
        logits = ops.matmul_nt(o.view(b, -1), head, workspace=gws)
        return serving.sample(logits, u, temp, topk, topp, workspace=ws2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok, lp = step()
    rng = np.random.RandomState(1)
    for turn in range(6):
        c = rng.randint(1, cap, b)
        order, at = rng.permutation(pool), 0
        table = np.full((b, cap // PAGE), -1)
        for s in range(b):
            need = -(-c[s] // PAGE)
            table[s, :need] = order[at:at + need]
            at += need
        if turn == 3:
            table[2] = -1  # an idle slot of a padded batch
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        ctx.copy_(_i32(c, dev))
        pages.copy_(_i32(table, dev))
        u.copy_(torch.rand(b, generator=g))
        temp.copy_(torch.tensor([0.0 if rng.rand() < 0.3 else 0.9 for _ in range(b)]))
        topk.copy_(_i32(rng.choice([0, 1, 40], b), dev))
        topp.copy_(torch.tensor(rng.choice([1.0, 0.9], b), dtype=torch.float32))
        before = k.clone(), v.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (q, o, tok, lp, k, v)]
        k.copy_(before[0])
        v.copy_(before[1])
        etok, elp = step()
        torch.cuda.synchronize()
        for x, y in zip(got, (q, o, etok, elp, k, v)):
            assert torch.equal(x, y)


def test_calls_on_a_stream_of_their_own(dev):
    """Two streams at once, each with its workspaces, against the default stream's results."""
    b = ref.Batch([1, 30, 1], [300, 200, 2000], 2, 128, 16, dev)
    arrays = b.device()
    g = torch.Generator().manual_seed(4)
    qs = [torch.randn((b.tokens, 4, 128), generator=g).half().to(dev) for _ in range(2)]
    xs = [torch.randn((3, 60000), generator=g).to(dev) for _ in range(2)]
    u = torch.rand(3, generator=g).to(dev)
    k50 = torch.full((3,), 50, dtype=torch.int32, device=dev)

    def both(i):
        return (serving.paged_attention(qs[i], *arrays, 30, 2000, 0.1), *serving.sample(xs[i], u, top_k=k50))

    want = [both(0), both(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = both(i)
    torch.cuda.synchronize()
    for w, x in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(w, x))


def test_the_binding_and_the_python_path_make_the_same_calls(dev, monkeypatch):
    """Every call here is one that the binding takes; through Python it gives the same bits, into new outputs and
    given ones."""
    b = ref.Batch([40, 1, 3], [90, 300, 70], 2, 64, 16, dev)
    g = torch.Generator().manual_seed(3)
    k, v, start, ctx, table = b.device()
    heads, rows = 4, b.tokens
    qkv = torch.randn((rows, (heads + 4) * 64), generator=g).half().to(dev)
    cos, sin = (torch.from_numpy(t).to(dev) for t in serving.rope_table_scaled(400, 64, 1e4))
    norms = (torch.rand((2, 64), generator=g) + 0.5).to(dev)
    pos = torch.arange(rows, dtype=torch.int32, device=dev)
    logits = (torch.randn((5, 20000), generator=g) * 3).to(dev)
    u, t, p, m = (torch.rand(5, generator=g).to(dev) for _ in range(4))
    top = torch.tensor([0, 1, 40, 5, 0], dtype=torch.int32, device=dev)
    heads_of = qkv.view(rows, heads + 4, 64)
    zeros = lambda *s: torch.zeros(s, dtype=torch.float16, device=dev)  # noqa: E731
    byte = torch.empty(1 << 22, dtype=torch.uint8, device=dev)
    calls = [
        ("rotary", lambda: serving.rotary(heads_of[:, 1:5], cos, sin, pos)),
        ("rotary", lambda: serving.rotary(heads_of[:, :6].float(), cos, sin, pos, True, torch.zeros((rows, 6, 64), device=dev))),
        ("qk_rope_append_paged", lambda: serving.qk_rope_append_paged(qkv, cos, sin, k, v, start, ctx, table, heads)),
        ("qk_rope_append_paged", lambda: serving.qk_rope_append_paged(qkv.float(), cos, sin, k, v, start, ctx, table, heads, norms,
                                                                      1e-5, True, zeros(rows, heads, 64))),
        ("paged_attention", lambda: serving.paged_attention(heads_of[:, :4], k, v, start, ctx, table, 40, 300, 0.125)),
        ("paged_attention", lambda: serving.paged_attention(heads_of[:, :4], k, v, start, ctx, table, 40, 5000, 1, 50,
                                                            zeros(rows, heads, 64), byte)),
        ("sample", lambda: serving.sample(logits, u, t, top, p, m)),
        ("sample", lambda: serving.sample(logits.half()[:, :9000], u, workspace=byte)),
    ]
    for name, call in calls:
        taken, real = [], getattr(serving._serving, name)

        def watched(*args, real=real, taken=taken):
            taken.append(real(*args))
            return taken[-1]

        with monkeypatch.context() as mp:
            mp.setattr(serving._serving, name, watched)
            got = call()
            cache = k.clone(), v.clone()
        assert taken[0] is not None, name
        with monkeypatch.context() as mp:
            mp.setattr(serving._serving, name, lambda *args: None)
            want = call()
        for x, y in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
            assert x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y), name
        assert all(torch.equal(x.nan_to_num(9.0), y.nan_to_num(9.0)) for x, y in zip(cache, (k, v)))
    out = zeros(rows, heads, 64)
    assert serving.paged_attention(heads_of[:, :4], k, v, start, ctx, table, 40, 300, out=out) is out


def test_captured_long_rows_and_split_contexts(dev):
    """The calls of several launches in two graphs, each with a workspace of its own, replayed in turn while logits,
    settings, lengths and pages change, with eager calls between: every replay against the eager result."""
    g = torch.Generator().manual_seed(5)
    rows, vocab, heads = 5, 40000, 8
    x, u = torch.zeros((rows, vocab), device=dev), torch.zeros(rows, device=dev)
    t, p = torch.ones(rows, device=dev), torch.ones(rows, device=dev)
    k = torch.zeros(rows, dtype=torch.int32, device=dev)
    b = ref.Batch([1, 40, 1, 2], [900, 700, 64, 1500], 4, 64, 16, dev)
    kp, vp, start, ctx, table = b.device()
    q = torch.zeros((b.tokens, heads, 64), dtype=torch.float16, device=dev)
    need = serving.paged_attention_workspace_bytes(b.tokens, 4, heads, 4, 64, 40, 1500), serving.sample_workspace_bytes(rows, vocab)
    assert min(need) > 0
    graphs = []
    for _ in range(2):
        ws = [torch.full((n,), 255, dtype=torch.uint8, device=dev) for n in need]
        serving.sample(x, u, t, k, p, workspace=ws[1])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = serving.sample(x, u, t, k, p, workspace=ws[1]), serving.paged_attention(q, kp, vp, start, ctx, table, 40, 1500, 0.1,
                                                                                           workspace=ws[0])
        graphs.append((graph, out, ws))
    for i in range(6):
        x.copy_(torch.randn((rows, vocab), generator=g) * 3)
        u.copy_(torch.rand(rows, generator=g))
        t.copy_(torch.tensor([0.0, 1.0, 0.7, 1.3, 0.9]).roll(i))
        k.copy_(torch.tensor([0, 50, 0, 3000, 1], dtype=torch.int32).roll(2 * i))
        p.copy_(torch.tensor([1.0, 0.9, 0.5, 1.0, 0.99]).roll(3 * i))
        q.copy_((torch.randn(q.shape, generator=g)).half())
        ctx.copy_(torch.tensor([900 - 100 * i, 700 - 130 * i, 64 - i, 1500 - 7 * i], dtype=torch.int32))
        graph, ((token, logprob), o), _ = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        (want, lp), wo = serving.sample(x, u, t, k, p), serving.paged_attention(q, kp, vp, start, ctx, table, 40, 1500, 0.1)
        assert torch.equal(token, want) and torch.equal(logprob, lp) and torch.equal(o, wo), i
