"""The serving entry points on the CPU: scaled RoPE tables against their formulas, refusals before any
device work, workspace sizes."""
import ctypes

import numpy as np
import pytest
import torch

from dtts import DttsError, _lib, ops, serving


def _freqs(rot, base, scaling, factor, original, fast=32.0, slow=1.0):
    i = np.arange(0, rot, 2, dtype=np.float64) / rot
    f = base ** -i
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "ntk":
        return (base * factor ** (rot / (rot - 2))) ** -i, 1.0
    if scaling == "yarn":
        # a pair makes original * f / 2 pi turns; the ramp runs between the (rounded outwards) pair indices
        # where that is `fast` and `slow`
        def index(turns):
            return rot / 2 * np.log(original / (2 * np.pi * turns)) / np.log(base)
        low, high = max(np.floor(index(fast)), 0), min(np.ceil(index(slow)), rot - 1)
        r = np.clip((np.arange(rot // 2) - low) / max(high - low, 1e-3), 0, 1)
        return f / factor * r + f * (1 - r), 0.1 * np.log(factor) + 1
    return f, 1.0


@pytest.mark.parametrize("rot,base,scaling,factor", [(128, 1e6, "none", 1.0), (64, 1e4, "linear", 4.0), (128, 1e4, "ntk", 8.0),
                                                     (128, 1e6, "yarn", 4.0), (32, 1e4, "yarn", 16.0), (2, 1e4, "linear", 1.0)])
def test_scaled_table(rot, base, scaling, factor):
    length, original = 3001, 750
    c, s = serving.rope_table_scaled(length, rot, base, scaling, factor, original)
    f, m = _freqs(rot, base, scaling, factor, original)
    a = np.arange(length, dtype=np.float64)[:, None] * f
    # one f32 rounding of a value up to m, after angles off by a few f64 roundings of up to `length` radians
    tol = m * (2.0 ** -24 + length * 2.0 ** -50)
    assert np.max(np.abs(c - np.cos(a) * m)) <= tol and np.max(np.abs(s - np.sin(a) * m)) <= tol


def test_unscaled_table_is_the_plain_one():
    a, b = serving.rope_table_scaled(517, 64, 1e6), ops.rope_table_f32(517, 64, 1e6)
    assert all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(a, b))


def test_yarn_keeps_fast_pairs_and_divides_slow_ones():
    args = (2000, 128, 1e4, "yarn", 8.0, 4096)
    c, s = serving.rope_table_scaled(*args, attn_factor=1.0)
    plain = serving.rope_table_scaled(2000, 128, 1e4)
    slow = serving.rope_table_scaled(2000, 128, 1e4, "linear", 8.0)
    assert np.array_equal(c[:, 0], plain[0][:, 0]) and np.array_equal(s[:, -1], slow[1][:, -1])


@pytest.mark.parametrize("kw,match", [
    (dict(rot_dim=7), "bad arguments"), (dict(base=1.0), "bad arguments"), (dict(scaling="linear", factor=0.5), "factor"),
    (dict(scaling="linear", factor=float("nan")), "factor"), (dict(scaling="ntk", rot_dim=2, factor=2.0), "more than one pair"),
    (dict(scaling="yarn", factor=2.0), "original_len"), (dict(scaling="yarn", factor=2.0, original_length=8, beta_fast=1.0), "beta_fast"),
    (dict(scaling="cubic"), "unknown scaling"),
])
def test_scaled_table_refusals(kw, match):
    args = dict(length=4, rot_dim=8, base=1e4)
    args.update(kw)
    with pytest.raises(DttsError, match=match):
        serving.rope_table_scaled(**args)


P = ctypes.c_void_p(4096)  # an aligned address that no refused call reads


def _refused(fn, match, *args):
    rc = getattr(_lib.lib(), fn)(*args)
    assert rc == -1 and match in _lib.lib().dtts_last_error().decode(), (rc, _lib.lib().dtts_last_error())


def _rotary(x=P, cos=P, sin=P, pos=P, y=P, rows=4, heads=2, hd=64, rot=64, layout=0, xs=128, ys=128, table=16):
    return x, cos, sin, pos, y, rows, heads, hd, rot, layout, xs, ys, table, None


@pytest.mark.parametrize("kw,match", [
    (dict(rows=-1), "bad shape"), (dict(heads=0), "bad shape"), (dict(table=0), "bad shape"), (dict(rot=63), "rotated dimensions"),
    (dict(rot=66), "rotated dimensions"), (dict(rot=0), "rotated dimensions"), (dict(layout=2), "unknown layout"),
    (dict(xs=127), "row strides"), (dict(ys=0), "row strides"), (dict(pos=None), "null pointer"), (dict(ys=160), "equal row strides"),
    (dict(x=ctypes.c_void_p(4098)), "misaligned"), (dict(rows=1 << 31), "too many rows"),
    # sizes whose products pass 64 bits
    (dict(rows=1 << 62), "too many rows"), (dict(y=ctypes.c_void_p(8192), heads=1 << 19, hd=1 << 19, rot=2, xs=1 << 40, ys=1 << 40), "too many rows"),
    (dict(y=ctypes.c_void_p(8196), layout=1, hd=65, rot=2, xs=130, ys=130), "interleaved pairs"),
])
def test_rotary_refusals(kw, match):
    _refused("dtts_rotary_f32", match, *_rotary(**kw))


def test_empty_calls_are_no_ops():
    lib = _lib.lib()
    assert lib.dtts_rotary_f16(*_rotary(rows=0, x=None)) == 0
    assert lib.dtts_qk_rope_append_paged_f32(*_append(tokens=0, qkv=None)) == 0
    assert lib.dtts_qk_rope_append_paged_f16(*_append(b=0, qkv=None)) == 0
    assert lib.dtts_paged_attention_f16(*_attention(tokens=0, q=None)) == 0
    assert lib.dtts_sample_f32(*_sample(rows=0, logits=None)) == 0


def _append(qkv=P, norms=None, cos=P, sin=P, start=P, ctx=P, table=P, q=P, k=P, v=P, tokens=3, b=2, heads=4, n_kv=2, hd=64,
            rot=64, layout=0, page=16, n_pages=8, max_pages=4, stride=2048, table_len=64):
    return (qkv, norms, cos, sin, start, ctx, table, q, k, v, tokens, b, heads, n_kv, hd, rot, layout, page, n_pages, max_pages,
            stride, table_len, 1e-6, None)


PAGED = [(dict(tokens=-1), "bad shape"), (dict(b=-1), "bad shape"), (dict(n_kv=0), "bad shape"), (dict(n_pages=0), "bad shape"),
         (dict(hd=96), "head_dim"), (dict(page=24), "power of two"), (dict(page=8), "power of two"), (dict(stride=2047), "page_stride"),
         (dict(stride=2052), "page_stride"), (dict(stride=1 << 33), "page_stride"), (dict(n_kv=1 << 60), "too many"),
         (dict(max_pages=1 << 62), "too many"), (dict(max_pages=(1 << 26) + 1), "too many"), (dict(b=1 << 17), "too many"),
         (dict(max_pages=1 << 28), "too many"),
         (dict(tokens=1 << 24), "too many"), (dict(start=None), "null pointer"), (dict(k=ctypes.c_void_p(4100)), "misaligned")]


@pytest.mark.parametrize("kw,match", PAGED + [
    (dict(heads=0), "heads"), (dict(rot=12), "rotated dimensions"), (dict(rot=72), "rotated dimensions"), (dict(layout=-1), "unknown layout"),
    (dict(table_len=0), "table"), (dict(cos=ctypes.c_void_p(4104)), "misaligned"), (dict(norms=ctypes.c_void_p(4104)), "misaligned"),
    (dict(), "may not replace qkv"),
])
def test_append_refusals(kw, match):
    for fn in ("dtts_qk_rope_append_paged_f32", "dtts_qk_rope_append_paged_f16"):
        _refused(fn, match, *_append(**kw))


def _attention(q=P, k=P, v=P, start=P, ctx=P, table=P, out=ctypes.c_void_p(8192), tokens=3, b=2, heads=4, n_kv=2, hd=64, page=16,
               n_pages=8, max_pages=4, stride=2048, q_stride=256, max_q=2, max_context=40, window=0, ws=None, ws_bytes=0,
               scale=1.0):
    return (q, k, v, start, ctx, table, out, tokens, b, heads, n_kv, hd, page, n_pages, max_pages, stride, q_stride, max_q,
            max_context, window, scale, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,match", PAGED + [
    (dict(heads=5), "heads over"), (dict(q_stride=255), "q_stride"), (dict(q_stride=260), "q_stride"), (dict(window=-1), "window"),
    (dict(max_q=0), "max_q"), (dict(max_context=0), "max_context"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=3e38), "scale"),
    (dict(tokens=(1 << 24) - 1, heads=16, n_kv=16, stride=16384, q_stride=1024), "too many rows"), (dict(out=P), "may not be the queries"),
    (dict(out=ctypes.c_void_p(8200)), "misaligned"),
    (dict(max_context=60000, ws=ctypes.c_void_p(4100), ws_bytes=1 << 30), "misaligned workspace"),
])
def test_attention_refusals(kw, match):
    _refused("dtts_paged_attention_f16", match, *_attention(**kw))


def test_attention_workspace_sizes():
    f = serving.paged_attention_workspace_bytes
    assert f(48, 48, 16, 8, 128, 1, 100) == 0  # one chunk
    assert f(1, 1, 16, 8, 128, 1, 65536) >= 2 * 16 * 128 * 4
    assert f(1, 1, 16, 8, 128, 1, 65536, window=100) <= f(1, 1, 16, 8, 128, 1, 65536)
    assert 0 < f(1, 1, 16, 8, 128, 1, (1 << 31) - 1) < 1 << 30  # a hint past every table
    assert f(0, 1, 16, 8, 128, 1, 65536) == 0 and f(4, 4, 15, 8, 128, 1, 65536) == 0 and f(-1, 1, 16, 8, 128, 1, 10) == 0


def test_sample_workspace_sizes():
    f = serving.sample_workspace_bytes
    assert f(1, 2048) == 0 and f(4000, 131072) == 0  # one workgroup a row
    assert 0 < f(1, 131072) == f(3, 131072) / 3
    assert f(0, 131072) == 0 and f(-1, 131072) == 0 and f(1, 1 << 21) == 0


def _sample(logits=P, t=None, k=None, p=None, m=None, u=P, token=P, logprob=None, rows=2, vocab=100, stride=100, ws=None, n=0):
    return logits, t, k, p, m, u, token, logprob, rows, vocab, stride, ws, n, None


@pytest.mark.parametrize("kw,match", [
    (dict(rows=-1), "bad shape"), (dict(rows=1 << 20), "bad shape"), (dict(vocab=0), "bad shape"),
    (dict(vocab=(1 << 20) + 1, stride=1 << 21), "vocabulary"),
    (dict(stride=99), "row stride"), (dict(u=None), "null pointer"), (dict(token=None), "null pointer"),
    (dict(logits=ctypes.c_void_p(4097)), "misaligned"), (dict(k=ctypes.c_void_p(4098)), "misaligned"),
])
def test_sample_refusals(kw, match):
    for fn in ("dtts_sample_f32", "dtts_sample_f16"):
        _refused(fn, match, *_sample(**kw))


def test_python_layer_refuses_host_tensors():
    x = torch.zeros((2, 2, 64))
    c = torch.zeros((4, 32))
    with pytest.raises(DttsError, match="on the device"):
        serving.rotary(x, c, c, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(DttsError, match="on the device"):
        serving.sample(torch.zeros((2, 9)), torch.zeros(2))
    with pytest.raises(DttsError, match="f16"):
        serving.paged_attention(x, x, x, x, x, x, 1, 1)


def test_the_binding_takes_no_wrong_call():
    """Anything that is not a right call on the current device is left to the Python path."""
    b, x = serving._serving, torch.zeros(2, 3, 64)
    i = torch.zeros(2, dtype=torch.int32)
    assert b.rotary(x, x[0], x[0], i, False, None) is None  # not on a GPU
    assert b.rotary(None, 1, "2", [], False, None) is None
    assert b.qk_rope_append_paged(x, *[i] * 7, 4, None, 1e-6, False, None) is None
    assert b.paged_attention(x, *[i] * 5, 1, 1, 1.0, 0, None, None) is None
    assert b.sample(x[0], i, None, None, None, None, None) is None
    for f in (b.rotary, b.qk_rope_append_paged, b.paged_attention, b.sample):
        with pytest.raises(TypeError, match="arguments expected"):
            f(x)
