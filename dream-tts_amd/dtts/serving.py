"""What a server of many requests calls beside the ops of ``dtts.ops``: rotary positions of every
layout and scaling, a paged KV cache's write and attention over ragged batches, and sampling.

A step of a batch is: project to qkv, ``qk_rope_append_paged`` (queries turned, keys and values into
their pages), ``paged_attention``, the output projection, and after the last layer logits to
``sample``. Lengths, positions, page tables and sampling settings are device tensors, so a step
captured into a graph is replayed while they change. Outputs are allocated unless given.

Every tensor of a call is on one device; the work goes to that device's current stream.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import DttsError, call, lib, ptr, stream_handle

_F16, _F32, _I32 = torch.float16, torch.float32, torch.int32
_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}


def _check(name, device, **tensors):
    """what=(tensor, dtypes): a contiguous tensor of one of them, on `device`."""
    for what, (t, dtypes) in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise DttsError(f"{name}: {what} must be a tensor")
        if t.device != device or device.type != "cuda":
            raise DttsError(f"{name}: {what} must be on the device ({t.device}, {device})")
        if t.dtype not in dtypes:
            raise DttsError(f"{name}: {what} dtype {t.dtype} not in {dtypes}")
        if not t.is_contiguous():
            raise DttsError(f"{name}: {what} must be contiguous")


def _enqueue(fn, device, *args):
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            call(fn, *args, stream_handle(device))
    else:
        call(fn, *args, stream_handle(device))


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


def _tables(name, cos, sin):
    if cos.dim() != 2 or cos.shape != sin.shape:
        raise DttsError(f"{name}: cos {tuple(cos.shape)} and sin {tuple(sin.shape)} must be [positions, rot_dim / 2]")
    return cos.shape


def _rows(name, t, what):
    """[rows, heads, D], each row contiguous: the elements between rows."""
    if t.dim() != 3 or t.stride(2) != 1 or t.stride(1) != t.shape[2]:
        raise DttsError(f"{name}: {what} must be [rows, heads, D] with contiguous rows, got {tuple(t.shape)} {t.stride()}")
    width = t.shape[1] * t.shape[2]
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), width)


def rotary(x, cos, sin, pos, interleaved=False, out=None):
    """x [rows, heads, D] (f32 or f16; rows may be strided, as a slice of qkv is) with the first
    2 * cos.shape[1] dimensions of each head turned by its row's position pos [rows] int32 (device). A
    position outside the tables is padding: that row of `out` is left as it was (of a new one: unset).
    out may be x."""
    name = "rotary"
    if not isinstance(x, torch.Tensor) or x.dtype not in (_F32, _F16):
        raise DttsError(f"{name}: x must be an f32 or f16 tensor")
    xs = _rows(name, x, "x")
    _check(name, x.device, cos=(cos, (_F32,)), sin=(sin, (_F32,)), pos=(pos, (_I32,)))
    n, half = _tables(name, cos, sin)
    rows, heads, hd = x.shape
    if pos.numel() != rows:
        raise DttsError(f"{name}: {pos.numel()} positions for {rows} rows")
    if out is None:
        out = torch.empty((rows, heads, hd), dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise DttsError(f"{name}: out {tuple(out.shape)} {out.dtype} for x {tuple(x.shape)} {x.dtype}")
    ys = _rows(name, out, "out")
    _enqueue("dtts_rotary_f32" if x.dtype == _F32 else "dtts_rotary_f16", x.device, ptr(x), ptr(cos), ptr(sin), ptr(pos),
             ptr(out), rows, heads, hd, 2 * half, int(interleaved), xs, ys, n)
    return out


# ---------------------------------------------------------------- the paged cache

def _paged(name, k_pages, v_pages, q_start, context, pages):
    """The cache's and the batch's sizes: pages [n_pages, n_kv, page, D], each contiguous."""
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.stride() != v_pages.stride():
        raise DttsError(f"{name}: k pages {tuple(k_pages.shape)} and v pages {tuple(v_pages.shape)}")
    if k_pages.dtype != _F16 or v_pages.dtype != _F16:
        raise DttsError(f"{name}: pages are f16")
    n_pages, n_kv, page, hd = k_pages.shape
    st = k_pages.stride()
    if st[1:] != (page * hd, hd, 1):
        raise DttsError(f"{name}: a page must be contiguous, got strides {st}")
    if pages.dim() != 2 or pages.shape[0] != context.numel() or q_start.numel() != pages.shape[0] + 1:
        raise DttsError(f"{name}: page table {tuple(pages.shape)}, {context.numel()} contexts, {q_start.numel()} starts")
    return pages.shape[0], n_kv, hd, page, n_pages, pages.shape[1], max(st[0], n_kv * page * hd) if n_pages == 1 else st[0]


def qk_rope_append_paged(qkv, cos, sin, k_pages, v_pages, q_start, context, pages, heads, norms=None, eps=1e-6,
                         interleaved=False, out=None):
    """QK-norm (norms [2, D] f32, or None), rotary positions and the write of a ragged batch's new keys and
    values: qkv [tokens, (heads + 2 n_kv) D] f32 or f16 -> queries [tokens, heads, D] f16; k_pages and
    v_pages [n_pages, n_kv, page, D] f16 are written in place. q_start [b + 1], context [b] (new tokens
    included) and pages [b, max_pages] are int32; see dtts.h for what each selects. Rows of `out` that
    belong to no sequence are left as they were."""
    name = "qk_rope_append_paged"
    dev = k_pages.device
    _check(name, dev, qkv=(qkv, (_F32, _F16)), cos=(cos, (_F32,)), sin=(sin, (_F32,)), q_start=(q_start, (_I32,)),
           context=(context, (_I32,)), pages=(pages, (_I32,)))
    if v_pages.device != dev:
        raise DttsError(f"{name}: v_pages must be on the device ({v_pages.device}, {dev})")
    n, half = _tables(name, cos, sin)
    b, n_kv, hd, page, n_pages, max_pages, stride = _paged(name, k_pages, v_pages, q_start, context, pages)
    if qkv.dim() != 2 or qkv.shape[1] != (heads + 2 * n_kv) * hd:
        raise DttsError(f"{name}: qkv {tuple(qkv.shape)} is not [tokens, ({heads} + 2 * {n_kv}) * {hd}]")
    if norms is not None:
        _check(name, dev, norms=(norms, (_F32,)))
        if norms.numel() != 2 * hd:
            raise DttsError(f"{name}: norms {tuple(norms.shape)} is not [2, {hd}]")
    tokens = qkv.shape[0]
    if out is None:
        out = torch.empty((tokens, heads, hd), dtype=_F16, device=dev)
    else:
        _check(name, dev, out=(out, (_F16,)))
        if out.numel() != tokens * heads * hd:
            raise DttsError(f"{name}: out {tuple(out.shape)} is not [{tokens}, {heads}, {hd}]")
    _enqueue("dtts_qk_rope_append_paged_f32" if qkv.dtype == _F32 else "dtts_qk_rope_append_paged_f16", dev, ptr(qkv),
             ptr(norms), ptr(cos), ptr(sin), ptr(q_start), ptr(context), ptr(pages), ptr(out), ptr(k_pages), ptr(v_pages),
             tokens, b, heads, n_kv, hd, 2 * half, int(interleaved), page, n_pages, max_pages, stride, n, float(eps))
    return out


def paged_attention_workspace_bytes(tokens, b, heads, n_kv, head_dim, max_q, max_context, window=0):
    """Workspace bytes paged_attention splits contexts over workgroups with."""
    return int(lib().dtts_paged_attention_workspace_bytes(tokens, b, heads, n_kv, head_dim, max_q, max_context, window))


def paged_attention(q, k_pages, v_pages, q_start, context, pages, max_q, max_context, scale=1.0, window=0, out=None,
                    workspace=None):
    """Attention of a ragged batch's new tokens over their pages, their own keys included: q [tokens, heads,
    D] f16 (rows may be strided) -> [tokens, heads, D] f16. Each token attends to its sequence's positions
    up to its own, the last `window` of them when set. max_q and max_context (the longest chunk and context)
    size the launch and never change what is computed. `workspace`: a device byte tensor of
    paged_attention_workspace_bytes (allocated when not given). Rows of `out` that belong to no sequence are
    left as they were; a token that sees no position gets zeros."""
    name = "paged_attention"
    dev = q.device
    if q.dtype != _F16:
        raise DttsError(f"{name}: q must be f16")
    qs = _rows(name, q, "q")
    _check(name, dev, q_start=(q_start, (_I32,)), context=(context, (_I32,)), pages=(pages, (_I32,)))
    if k_pages.device != dev or v_pages.device != dev:
        raise DttsError(f"{name}: the pages must be on the device ({k_pages.device}, {v_pages.device}, {dev})")
    b, n_kv, hd, page, n_pages, max_pages, stride = _paged(name, k_pages, v_pages, q_start, context, pages)
    tokens, heads, qd = q.shape
    if qd != hd:
        raise DttsError(f"{name}: q {tuple(q.shape)} over pages of head_dim {hd}")
    if out is None:
        out = torch.empty((tokens, heads, hd), dtype=_F16, device=dev)
    else:
        _check(name, dev, out=(out, (_F16,)))
        if out.numel() != tokens * heads * hd:
            raise DttsError(f"{name}: out {tuple(out.shape)} is not [{tokens}, {heads}, {hd}]")
    if workspace is None:
        need = paged_attention_workspace_bytes(tokens, b, heads, n_kv, hd, max_q, max_context, window)
        workspace = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _enqueue("dtts_paged_attention_f16", dev, ptr(q), ptr(k_pages), ptr(v_pages), ptr(q_start), ptr(context), ptr(pages),
             ptr(out), tokens, b, heads, n_kv, hd, page, n_pages, max_pages, stride, qs, max_q, max_context, window,
             float(scale), ptr(workspace), workspace.numel() if workspace is not None else 0)
    return out


# ---------------------------------------------------------------- sampling

def sample_workspace_bytes(rows, vocab):
    """Workspace bytes sample splits a long row over workgroups with."""
    return int(lib().dtts_sample_workspace_bytes(rows, vocab))


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, workspace=None):
    """One token per row of logits [rows, vocab] (f32 or f16; rows may be strided) from the uniform random
    numbers u [rows] in [0, 1): (tokens int32 [rows], log-probabilities f32 [rows] under the distribution
    sampled from). temperature, top_p, min_p f32 [rows] and top_k int32 [rows] are each row's settings or
    None; temperature 0 takes the largest logit, top_k 0, top_p 1 and min_p 0 filter nothing. A row without
    a finite (or +inf) logit gives token -1."""
    name = "sample"
    if not isinstance(logits, torch.Tensor) or logits.dtype not in (_F32, _F16) or logits.dim() != 2:
        raise DttsError(f"{name}: logits must be an f32 or f16 tensor [rows, vocab]")
    rows, vocab = logits.shape
    if logits.stride(1) != 1 and vocab > 1:
        raise DttsError(f"{name}: a row of logits must be contiguous, got strides {logits.stride()}")
    dev = logits.device
    _check(name, dev, u=(u, (_F32,)))
    for what, t, dtype in (("temperature", temperature, _F32), ("top_k", top_k, _I32), ("top_p", top_p, _F32),
                           ("min_p", min_p, _F32)):
        if t is not None:
            _check(name, dev, **{what: (t, (dtype,))})
            if t.numel() != rows:
                raise DttsError(f"{name}: {t.numel()} of {what} for {rows} rows")
    if u.numel() != rows:
        raise DttsError(f"{name}: {u.numel()} random numbers for {rows} rows")
    token = torch.empty(rows, dtype=_I32, device=dev)
    logprob = torch.empty(rows, dtype=_F32, device=dev)
    if workspace is None:
        need = sample_workspace_bytes(rows, vocab)
        workspace = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _enqueue("dtts_sample_f32" if logits.dtype == _F32 else "dtts_sample_f16", dev, ptr(logits), ptr(temperature), ptr(top_k),
             ptr(top_p), ptr(min_p), ptr(u), ptr(token), ptr(logprob), rows, vocab,
             logits.stride(0) if rows > 1 else max(logits.stride(0), vocab), ptr(workspace),
             workspace.numel() if workspace is not None else 0)
    return token, logprob
