"""What a server of many requests calls beside the ops of ``dtts.ops``: rotary positions of every
layout and scaling, a paged KV cache's write and attention over ragged batches, and sampling.

A step of a batch is: project to qkv, ``qk_rope_append_paged`` (queries turned, keys and values into
their pages), ``paged_attention``, the output projection, and after the last layer logits to
``sample``. Lengths, positions, page tables and sampling settings are device tensors, so a step
captured into a graph is replayed while they change. Outputs are allocated unless given.

Every tensor of a call is on one device; the work goes to that device's current stream.

A right call on the current device is checked and enqueued by ``_serving`` (csrc/serving_py.cpp), since
reading ten tensors' sizes and addresses in Python takes longer than the work. It returns None for any
other, and the Python below makes the call or says what is wrong with it. Where the binding was built
for another torch, Python makes all of them (and a warning says so).
"""
from __future__ import annotations

import ctypes
import functools
import types
import warnings

import torch

from ._lib import DttsError, call, lib

try:
    from . import _serving
except ImportError as e:
    warnings.warn(f"dtts/_serving.so is not built for this torch ({e}): calls of dtts.serving take some microseconds longer; "
                  "run dream-tts_amd/build.py", RuntimeWarning)
    _serving = types.SimpleNamespace(**dict.fromkeys(("rotary", "qk_rope_append_paged", "paged_attention", "sample"),
                                                     lambda *args: None))

_F16, _F32, _I32 = torch.float16, torch.float32, torch.int32
_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}
_Tensor = torch.Tensor


def _need(name, device, what, t, dtypes, contiguous=True):
    """Raises unless t is a (contiguous) tensor of one of dtypes on GPU number `device`. A step is a few
    microseconds of GPU work, and so is each of these calls on the host: the callers pass their tensors
    through one condition that holds for all of a right call, and come here to say what is wrong."""
    if not isinstance(t, _Tensor):
        raise DttsError(f"{name}: {what} must be a tensor")
    if device < 0 or t.get_device() != device:
        raise DttsError(f"{name}: {what} must be on the device ({t.device}, GPU {device})")
    if t.dtype not in dtypes:
        raise DttsError(f"{name}: {what} dtype {t.dtype} not in {dtypes}")
    if contiguous and not t.is_contiguous():
        raise DttsError(f"{name}: {what} must be contiguous")


def _enqueue(fn, device, *args):
    """The call on GPU number `device`'s current stream (as the raw handle: building a Stream object takes
    longer than the launch)."""
    if device == torch._C._cuda_getDevice():
        status = getattr(lib(), fn)(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            status = getattr(lib(), fn)(*args, torch._C._cuda_getCurrentRawStream(device))
    if status != 0:
        raise DttsError(f"{fn} failed ({status}): {lib().dtts_last_error().decode(errors='replace')}")


# ---------------------------------------------------------------- rotary positions

def rope_table_scaled(length, rot_dim, base, scaling="none", factor=1.0, original_length=0, beta_fast=32.0,
                      beta_slow=1.0, attn_factor=0.0):
    """(cos, sin) numpy f32 [length, rot_dim / 2] on the host for contexts longer than the trained one:
    scaling "none", "linear", "ntk" or "yarn" (dtts_rope_table_scaled_f32)."""
    import numpy as np

    if scaling not in _SCALINGS:
        raise DttsError(f"rope_table_scaled: unknown scaling {scaling!r}")
    c = np.empty((length, rot_dim // 2), np.float32)
    s = np.empty((length, rot_dim // 2), np.float32)
    call("dtts_rope_table_scaled_f32", length, rot_dim, float(base), _SCALINGS[scaling], float(factor), original_length,
         float(beta_fast), float(beta_slow), float(attn_factor), ctypes.c_void_p(c.ctypes.data),
         ctypes.c_void_p(s.ctypes.data))
    return c, s


def _tables(name, device, cos, sin):
    if not (isinstance(cos, _Tensor) and isinstance(sin, _Tensor) and cos.dtype is _F32 and sin.dtype is _F32
            and cos.get_device() == device and sin.get_device() == device and cos.is_contiguous() and sin.is_contiguous()):
        _need(name, device, "cos", cos, (_F32,))
        _need(name, device, "sin", sin, (_F32,))
    n = cos.shape
    if len(n) != 2 or n != sin.shape:
        raise DttsError(f"{name}: cos {tuple(n)} and sin {tuple(sin.shape)} must be [positions, rot_dim / 2]")
    return n


def _rows(name, t, what):
    """[rows, heads, D] with contiguous rows: its sizes, and the elements between rows. The stride of a size of 1 is no
    one's: torch leaves any number there, also after contiguous()."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or stride[2] != 1 or (stride[1] != shape[2] and shape[1] != 1):
        raise DttsError(f"{name}: {what} must be [rows, heads, D] with contiguous rows, got {tuple(shape)} {stride}")
    return shape, stride[0] if shape[0] > 1 else shape[1] * shape[2]


def rotary(x, cos, sin, pos, interleaved=False, out=None):
    """x [rows, heads, D] (f32 or f16; rows may be strided, as a slice of qkv is) with the first
    2 * cos.shape[1] dimensions of each head turned by its row's position pos [rows] int32 (device). A
    position outside the tables is padding: that row of `out` is left as it was (of a new one: unset).
    out may be x, and otherwise shares no memory with it."""
    y = _serving.rotary(x, cos, sin, pos, interleaved, out)
    if y is not None:
        return y
    name = "rotary"
    if not isinstance(x, _Tensor) or (x.dtype is not _F32 and x.dtype is not _F16):
        raise DttsError(f"{name}: x must be an f32 or f16 tensor")
    dev = x.get_device()
    if dev < 0:
        _need(name, dev, "x", x, (x.dtype,), contiguous=False)
    (rows, heads, hd), xs = _rows(name, x, "x")
    n, half = _tables(name, dev, cos, sin)
    if not (isinstance(pos, _Tensor) and pos.dtype is _I32 and pos.get_device() == dev and pos.is_contiguous()):
        _need(name, dev, "pos", pos, (_I32,))
    if pos.numel() != rows:
        raise DttsError(f"{name}: {pos.numel()} positions for {rows} rows")
    if out is None:
        out = torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)
        ys = heads * hd
    else:
        _need(name, dev, "out", out, (x.dtype,), contiguous=False)
        if out.shape != x.shape:
            raise DttsError(f"{name}: out {tuple(out.shape)} for x {tuple(x.shape)}")
        ys = _rows(name, out, "out")[1]
    _enqueue("dtts_rotary_f32" if x.dtype is _F32 else "dtts_rotary_f16", dev, x.data_ptr(), cos.data_ptr(), sin.data_ptr(),
             pos.data_ptr(), out.data_ptr(), rows, heads, hd, 2 * half, 1 if interleaved else 0, xs, ys, n)
    return out


# ---------------------------------------------------------------- the paged cache

def _page_stride(name, t):
    """The elements between the pages of [n_pages, n_kv, page, D], each of them contiguous."""
    (n_pages, n_kv, page, hd), st = t.shape, t.stride()
    if st[3] != 1 or st[2] != hd or (st[1] != page * hd and n_kv != 1):
        raise DttsError(f"{name}: a page must be contiguous, got strides {st}")
    return st[0] if n_pages > 1 else n_kv * page * hd


def _paged(name, device, k_pages, v_pages, q_start, context, pages):
    """Checks the cache [n_pages, n_kv, page, D] (each page contiguous) and the batch's arrays: b, n_kv, D,
    page, n_pages, max_pages and the elements between pages."""
    tensors = (k_pages, v_pages, q_start, context, pages)
    for t in tensors:
        if not isinstance(t, _Tensor) or t.get_device() != device:
            break
    else:
        if (k_pages.dtype is _F16 and v_pages.dtype is _F16 and q_start.dtype is _I32 and context.dtype is _I32
                and pages.dtype is _I32 and q_start.is_contiguous() and context.is_contiguous() and pages.is_contiguous()):
            tensors = None
    if tensors is not None:
        for t, what, dtype in zip(tensors, ("k_pages", "v_pages", "q_start", "context", "pages"), (_F16, _F16, _I32, _I32, _I32)):
            _need(name, device, what, t, (dtype,), contiguous=dtype is _I32)
    shape = k_pages.shape
    if len(shape) != 4 or shape != v_pages.shape:
        raise DttsError(f"{name}: k pages {tuple(shape)} and v pages {tuple(v_pages.shape)}")
    stride = _page_stride(name, k_pages)
    if stride != _page_stride(name, v_pages):
        raise DttsError(f"{name}: k pages {k_pages.stride()} and v pages {v_pages.stride()} apart")
    n_pages, n_kv, page, hd = shape
    table = pages.shape
    if len(table) != 2 or table[0] != context.numel() or q_start.numel() != table[0] + 1:
        raise DttsError(f"{name}: page table {tuple(table)}, {context.numel()} contexts, {q_start.numel()} starts")
    return table[0], n_kv, hd, page, n_pages, table[1], stride


def _out(name, device, out, like, tokens, heads, hd):
    if out is None:
        if like.dtype is _F16 and like.dim() == 3 and like.is_contiguous():
            return torch.empty_like(like)  # the queries' own shape, in half the time
        return torch.empty((tokens, heads, hd), dtype=_F16, device=like.device)
    _need(name, device, "out", out, (_F16,))
    if out.numel() != tokens * heads * hd:
        raise DttsError(f"{name}: out {tuple(out.shape)} is not [{tokens}, {heads}, {hd}]")
    return out


def _bytes(name, device, workspace, need, like):
    """(tensor kept alive, address, bytes) of a call's workspace."""
    if workspace is None:
        if not need:
            return None, None, 0
        workspace = torch.empty(need, dtype=torch.uint8, device=like.device)
    else:
        _need(name, device, "workspace", workspace, (torch.uint8,))
    return workspace, workspace.data_ptr(), workspace.numel()


def qk_rope_append_paged(qkv, cos, sin, k_pages, v_pages, q_start, context, pages, heads, norms=None, eps=1e-6,
                         interleaved=False, out=None):
    """QK-norm (norms [2, D] f32, or None), rotary positions and the write of a ragged batch's new keys and
    values: qkv [tokens, (heads + 2 n_kv) D] f32 or f16 -> queries [tokens, heads, D] f16; k_pages and
    v_pages [n_pages, n_kv, page, D] f16 are written in place. q_start [b + 1], context [b] (new tokens
    included) and pages [b, max_pages] are int32; see dtts.h for what each selects. Rows of `out` that
    belong to no sequence are left as they were. `out` is no part of qkv, and the pages share no memory."""
    y = _serving.qk_rope_append_paged(qkv, cos, sin, k_pages, v_pages, q_start, context, pages, heads, norms, eps, interleaved, out)
    if y is not None:
        return y
    name = "qk_rope_append_paged"
    if not isinstance(qkv, _Tensor):
        raise DttsError(f"{name}: qkv must be a tensor")
    dev = qkv.get_device()
    f32 = qkv.dtype is _F32
    if dev < 0 or not (f32 or qkv.dtype is _F16) or not qkv.is_contiguous():
        _need(name, dev, "qkv", qkv, (_F32, _F16))
    b, n_kv, hd, page, n_pages, max_pages, stride = _paged(name, dev, k_pages, v_pages, q_start, context, pages)
    n, half = _tables(name, dev, cos, sin)
    size = qkv.shape
    if len(size) != 2 or size[1] != (heads + 2 * n_kv) * hd:
        raise DttsError(f"{name}: qkv {tuple(qkv.shape)} is not [tokens, ({heads} + 2 * {n_kv}) * {hd}]")
    if norms is not None:
        if not (isinstance(norms, _Tensor) and norms.dtype is _F32 and norms.get_device() == dev and norms.is_contiguous()):
            _need(name, dev, "norms", norms, (_F32,))
        if norms.numel() != 2 * hd:
            raise DttsError(f"{name}: norms {tuple(norms.shape)} is not [2, {hd}]")
    tokens = size[0]
    out = _out(name, dev, out, qkv, tokens, heads, hd)
    _enqueue("dtts_qk_rope_append_paged_f32" if f32 else "dtts_qk_rope_append_paged_f16", dev, qkv.data_ptr(),
             None if norms is None else norms.data_ptr(), cos.data_ptr(), sin.data_ptr(), q_start.data_ptr(),
             context.data_ptr(), pages.data_ptr(), out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), tokens, b, heads,
             n_kv, hd, 2 * half, 1 if interleaved else 0, page, n_pages, max_pages, stride, n, float(eps))
    return out


@functools.lru_cache(maxsize=4096)
def paged_attention_workspace_bytes(tokens, b, heads, n_kv, head_dim, max_q, max_context, window=0):
    """Workspace bytes paged_attention splits contexts over workgroups with."""
    return int(lib().dtts_paged_attention_workspace_bytes(tokens, b, heads, n_kv, head_dim, int(max_q), int(max_context),
                                                          int(window)))


def paged_attention(q, k_pages, v_pages, q_start, context, pages, max_q, max_context, scale=1.0, window=0, out=None,
                    workspace=None):
    """Attention of a ragged batch's new tokens over their pages, their own keys included: q [tokens, heads,
    D] f16 (rows may be strided) -> [tokens, heads, D] f16. Each token attends to its sequence's positions
    up to its own, the last `window` of them when set. max_q and max_context (the longest chunk and context)
    size the launch and never change what is computed. `workspace`: a device byte tensor of
    paged_attention_workspace_bytes (allocated when not given). Rows of `out` that belong to no sequence are
    left as they were; a token that sees no position gets zeros. `out` shares no memory with q."""
    y = _serving.paged_attention(q, k_pages, v_pages, q_start, context, pages, max_q, max_context, scale, window, out, workspace)
    if y is not None:
        return y
    name = "paged_attention"
    if not isinstance(q, _Tensor) or q.dtype is not _F16:
        raise DttsError(f"{name}: q must be an f16 tensor")
    dev = q.get_device()
    if dev < 0:
        _need(name, dev, "q", q, (_F16,), contiguous=False)
    (tokens, heads, qd), qs = _rows(name, q, "q")
    b, n_kv, hd, page, n_pages, max_pages, stride = _paged(name, dev, k_pages, v_pages, q_start, context, pages)
    if qd != hd:
        raise DttsError(f"{name}: q {tuple(q.shape)} over pages of head_dim {hd}")
    out = _out(name, dev, out, q, tokens, heads, hd)
    need = 0 if workspace is not None else paged_attention_workspace_bytes(tokens, b, heads, n_kv, hd, max_q, max_context, window)
    keep = ws = None
    ws_bytes = 0
    if need or workspace is not None:
        keep, ws, ws_bytes = _bytes(name, dev, workspace, need, q)
    _enqueue("dtts_paged_attention_f16", dev, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), q_start.data_ptr(),
             context.data_ptr(), pages.data_ptr(), out.data_ptr(), tokens, b, heads, n_kv, hd, page, n_pages, max_pages, stride,
             qs, int(max_q), int(max_context), int(window), float(scale), ws, ws_bytes)
    return out


# ---------------------------------------------------------------- sampling

@functools.lru_cache(maxsize=4096)
def sample_workspace_bytes(rows, vocab):
    """Workspace bytes sample splits a long row over workgroups with."""
    return int(lib().dtts_sample_workspace_bytes(rows, vocab))


def _setting(name, device, what, t, dtype, rows):
    if t is None:
        return None
    if not (isinstance(t, _Tensor) and t.dtype is dtype and t.get_device() == device and t.is_contiguous()):
        _need(name, device, what, t, (dtype,))
    if t.numel() != rows:
        raise DttsError(f"{name}: {t.numel()} of {what} for {rows} rows")
    return t.data_ptr()


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, workspace=None):
    """One token per row of logits [rows, vocab] (f32 or f16; rows may be strided) from the uniform random
    numbers u [rows] in [0, 1): (tokens int32 [rows], log-probabilities f32 [rows] under the distribution
    sampled from). temperature, top_p, min_p f32 [rows] and top_k int32 [rows] are each row's settings or
    None; temperature 0 takes the largest logit, top_k 0, top_p 1 and min_p 0 filter nothing. A row without
    a finite (or +inf) logit gives token -1. `workspace`: a device byte tensor of sample_workspace_bytes
    (allocated when not given)."""
    y = _serving.sample(logits, u, temperature, top_k, top_p, min_p, workspace)
    if y is not None:
        return y
    name = "sample"
    if not isinstance(logits, _Tensor) or (logits.dtype is not _F32 and logits.dtype is not _F16) or logits.dim() != 2:
        raise DttsError(f"{name}: logits must be an f32 or f16 tensor [rows, vocab]")
    rows, vocab = logits.shape
    stride = logits.stride()
    if stride[1] != 1 and vocab > 1:
        raise DttsError(f"{name}: a row of logits must be contiguous, got strides {stride}")
    dev = logits.get_device()
    if dev < 0:
        _need(name, dev, "logits", logits, (logits.dtype,), contiguous=False)
    if u is None:
        raise DttsError(f"{name}: u must be a tensor")
    pu = _setting(name, dev, "random numbers", u, _F32, rows)
    pt = _setting(name, dev, "temperature", temperature, _F32, rows)
    pk = _setting(name, dev, "top_k", top_k, _I32, rows)
    pp = _setting(name, dev, "top_p", top_p, _F32, rows)
    pm = _setting(name, dev, "min_p", min_p, _F32, rows)
    token = torch.empty(rows, dtype=_I32, device=logits.device)
    logprob = torch.empty_like(u) if u.dim() == 1 else torch.empty(rows, dtype=_F32, device=logits.device)
    need = sample_workspace_bytes(rows, vocab)
    keep = ws = None
    ws_bytes = 0
    if need or workspace is not None:
        keep, ws, ws_bytes = _bytes(name, dev, workspace, need, logits)
    _enqueue("dtts_sample_f32" if logits.dtype is _F32 else "dtts_sample_f16", dev, logits.data_ptr(), pt, pk, pp, pm, pu,
             token.data_ptr(), logprob.data_ptr(), rows, vocab, stride[0] if rows > 1 else max(stride[0], vocab), ws, ws_bytes)
    return token, logprob
