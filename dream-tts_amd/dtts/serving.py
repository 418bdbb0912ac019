"""What a server of many requests calls beside the ops of ``dtts.ops``: rotary positions of every
layout and scaling, a paged KV cache's write and attention over ragged batches (f16 or in 4 bits), its
pages' forks, claims, trims, moves and copies, and sampling.

A step of a batch is: project to qkv, ``qk_rope_append_paged`` (queries turned, keys and values into
their pages), ``paged_attention``, the output projection, and after the last layer logits to
``sample``. Before a step, ``claim_pages`` gives each sequence the pages that its new tokens go to. Lengths, positions,
page tables and sampling settings are device tensors, so a step captured into a graph is replayed while they change. Outputs
are allocated unless given.

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
    _serving = types.SimpleNamespace(**dict.fromkeys(
        ("rotary", "qk_rope_append_paged", "paged_attention", "sample", "unpack_pages", "fork_pages", "claim_pages", "trim_pages",
         "compact_pages", "copy_pages"), lambda *args: None))

_F16, _F32, _I32, _U8 = torch.float16, torch.float32, torch.int32, torch.uint8
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


def _cache(name, device, k_pages, v_pages):
    """Checks the cache's pages [n_pages, n_kv, page, D] f16 or [n_pages, n_kv, page, 5 D / 8] uint8 (each contiguous): n_kv, D,
    page, n_pages, the elements (bytes) between pages, and the bits of a value."""
    for t, what in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        if not isinstance(t, _Tensor) or device < 0 or t.get_device() != device or (t.dtype is not _F16 and t.dtype is not _U8):
            _need(name, device, what, t, (_F16, _U8), contiguous=False)
    shape = k_pages.shape
    if len(shape) != 4 or shape != v_pages.shape or k_pages.dtype is not v_pages.dtype:
        raise DttsError(f"{name}: k pages {tuple(shape)} {k_pages.dtype} and v pages {tuple(v_pages.shape)} {v_pages.dtype}")
    stride = _page_stride(name, k_pages)
    if stride != _page_stride(name, v_pages):
        raise DttsError(f"{name}: k pages {k_pages.stride()} and v pages {v_pages.stride()} apart")
    n_pages, n_kv, page, row = shape
    if k_pages.dtype is _F16:
        return n_kv, row, page, n_pages, stride, 16
    if row % 5:
        raise DttsError(f"{name}: rows of {row} bytes are not 5 D / 8")
    return n_kv, row * 8 // 5, page, n_pages, stride, 4


def _paged(name, device, k_pages, v_pages, q_start, context, pages):
    """Checks the cache and the batch's arrays: b, n_kv, D, page, n_pages, max_pages, the elements between pages and the bits of
    a value."""
    n_kv, hd, page, n_pages, stride, bits = _cache(name, device, k_pages, v_pages)
    for t, what in ((q_start, "q_start"), (context, "context"), (pages, "pages")):
        if not (isinstance(t, _Tensor) and t.dtype is _I32 and t.get_device() == device and t.is_contiguous()):
            _need(name, device, what, t, (_I32,))
    table = pages.shape
    if len(table) != 2 or table[0] != context.numel() or q_start.numel() != table[0] + 1:
        raise DttsError(f"{name}: page table {tuple(table)}, {context.numel()} contexts, {q_start.numel()} starts")
    return table[0], n_kv, hd, page, n_pages, table[1], stride, bits


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
    v_pages, [n_pages, n_kv, page, D] f16 or 4-bit pages [n_pages, n_kv, page, 5 D / 8] uint8, are written in place. q_start [b + 1], context [b] (new tokens
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
    b, n_kv, hd, page, n_pages, max_pages, stride, bits = _paged(name, dev, k_pages, v_pages, q_start, context, pages)
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
    _enqueue(f"dtts_qk_rope_append_paged_{'q4_' if bits == 4 else ''}{'f32' if f32 else 'f16'}", dev, qkv.data_ptr(),
             None if norms is None else norms.data_ptr(), cos.data_ptr(), sin.data_ptr(), q_start.data_ptr(),
             context.data_ptr(), pages.data_ptr(), out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), tokens, b, heads,
             n_kv, hd, 2 * half, 1 if interleaved else 0, page, n_pages, max_pages, stride, n, float(eps))
    return out


@functools.lru_cache(maxsize=4096)
def paged_attention_workspace_bytes(tokens, b, heads, n_kv, head_dim, max_q, max_context, window=0, sinks=0, bits=16):
    """Workspace bytes paged_attention splits contexts over workgroups with (bits: 16, or 4 for 4-bit pages)."""
    return int(lib().dtts_paged_attention_sinks_workspace_bytes(int(bits), tokens, b, heads, n_kv, head_dim, int(max_q),
                                                                int(max_context), int(window), int(sinks)))


def paged_attention(q, k_pages, v_pages, q_start, context, pages, max_q, max_context, scale=1.0, window=0, out=None,
                    workspace=None, sinks=0):
    """Attention of a ragged batch's new tokens over their pages (f16, or 4-bit ones as qk_rope_append_paged
    writes them), their own keys included: q [tokens, heads, D] f16 (rows may be strided) -> [tokens, heads,
    D] f16. Each token attends to its sequence's positions up to its own, when `window` is set to the last
    `window` of them and to the sequence's first `sinks` (whose keys stay turned by their own positions, as the append wrote
    them: a token is as far from them as its position says, not as its window does). max_q and max_context (the
    longest chunk and context) size the launch and never change what is computed. `workspace`: a device byte tensor
    of paged_attention_workspace_bytes (allocated when not given). Rows of `out` that belong to no sequence are left
    as they were; a token that sees no position gets zeros. `out` shares no memory with q."""
    y = _serving.paged_attention(q, k_pages, v_pages, q_start, context, pages, max_q, max_context, scale, window, out, workspace,
                                 sinks)
    if y is not None:
        return y
    name = "paged_attention"
    if not isinstance(q, _Tensor) or q.dtype is not _F16:
        raise DttsError(f"{name}: q must be an f16 tensor")
    dev = q.get_device()
    if dev < 0:
        _need(name, dev, "q", q, (_F16,), contiguous=False)
    (tokens, heads, qd), qs = _rows(name, q, "q")
    b, n_kv, hd, page, n_pages, max_pages, stride, bits = _paged(name, dev, k_pages, v_pages, q_start, context, pages)
    if qd != hd:
        raise DttsError(f"{name}: q {tuple(q.shape)} over pages of head_dim {hd}")
    out = _out(name, dev, out, q, tokens, heads, hd)
    need = 0 if workspace is not None else paged_attention_workspace_bytes(tokens, b, heads, n_kv, hd, max_q, max_context, window,
                                                                                      sinks, bits)
    keep = ws = None
    ws_bytes = 0
    if need or workspace is not None:
        keep, ws, ws_bytes = _bytes(name, dev, workspace, need, q)
    _enqueue("dtts_paged_attention", dev, bits, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), q_start.data_ptr(),
             context.data_ptr(), pages.data_ptr(), out.data_ptr(), tokens, b, heads, n_kv, hd, page, n_pages, max_pages, stride,
             qs, int(max_q), int(max_context), int(window), int(sinks), float(scale), ws, ws_bytes)
    return out


def unpack_pages(k_pages, v_pages, ids=None):
    """The values (k, v) [n, n_kv, page, D] f16 of 4-bit pages [n_pages, n_kv, page, 5 D / 8] uint8: of all of
    them, or of the pages ids [n] int32 (a row of a page table, say; an id outside the pool leaves its part unset).
    Slots that hold no position stand for whatever is there."""
    y = _serving.unpack_pages(k_pages, v_pages, ids)
    if y is not None:
        return y
    name = "unpack_pages"
    if not isinstance(k_pages, _Tensor):
        raise DttsError(f"{name}: k_pages must be a tensor")
    dev = k_pages.get_device()
    n_kv, hd, page, n_pages, stride, bits = _cache(name, dev, k_pages, v_pages)
    if bits != 4:
        raise DttsError(f"{name}: k_pages dtype {k_pages.dtype} not in ({_U8},)")
    if ids is not None:
        _need(name, dev, "ids", ids, (_I32,))
    n = n_pages if ids is None else ids.numel()
    k, v = (torch.empty((n, n_kv, page, hd), dtype=_F16, device=k_pages.device) for _ in range(2))
    _enqueue("dtts_unpack_pages_q4", dev, k_pages.data_ptr(), v_pages.data_ptr(), None if ids is None else ids.data_ptr(),
             k.data_ptr(), v.data_ptr(), n, n_kv, hd, page, n_pages, stride)
    return k, v


# ---------------------------------------------------------------- the cache's pages between steps

def _table(name, pages, refs, *more):
    """Checks a page table, its pages' counts and further int32 arrays (tensor, name, elements): the device."""
    if not isinstance(pages, _Tensor):
        raise DttsError(f"{name}: pages must be a tensor")
    dev = pages.get_device()
    for t, what in ((pages, "pages"), (refs, "refs"), *((t, what) for t, what, _ in more)):
        if not (isinstance(t, _Tensor) and t.dtype is _I32 and t.get_device() == dev and t.is_contiguous()) or dev < 0:
            _need(name, dev, what, t, (_I32,))
    if pages.dim() != 2 or refs.dim() != 1:
        raise DttsError(f"{name}: pages {tuple(pages.shape)} and refs {tuple(refs.shape)} must be [b, max_pages] and [n_pages]")
    for t, what, n in more:
        if n is not None and t.numel() != n:
            raise DttsError(f"{name}: {t.numel()} of {what} for a page table {tuple(pages.shape)}")
    return dev


def _empty_i32(n, like):
    return torch.empty(n, dtype=_I32, device=like.device)


def fork_pages(pages, refs, parent, out=None, workspace=None):
    """A table whose row i has the pages of row parent[i] (int32 [n]; none for a parent outside the table), and refs
    (int32 [n_pages], how many entries hold each page) brought up to it in place: forks and reorders sequences and
    frees those that no row takes over. `out`: None for a new table [n, max_pages], or `pages` itself for the
    change in place (through a workspace of as many bytes, allocated when not given)."""
    y = _serving.fork_pages(pages, refs, parent, out, workspace)
    if y is not None:
        return y
    name = "fork_pages"
    dev = _table(name, pages, refs, (parent, "parent", None))
    (b, m), n = pages.shape, parent.numel()
    if out is None:
        out = torch.empty((n, m), dtype=_I32, device=pages.device)
    else:
        _need(name, dev, "out", out, (_I32,))
        if out.shape != (n, m):
            raise DttsError(f"{name}: out {tuple(out.shape)} is not [{n}, {m}]")
    keep, ws, ws_bytes = _bytes(name, dev, workspace, 4 * b * m if out.data_ptr() == pages.data_ptr() else 0, pages)
    _enqueue("dtts_fork_pages", dev, pages.data_ptr(), refs.data_ptr(), parent.data_ptr(), out.data_ptr(), b, n, m, refs.numel(), ws,
             ws_bytes)
    return out


def claim_pages_workspace_bytes(b, max_pages, n_pages):
    return int(lib().dtts_claim_pages_workspace_bytes(b, max_pages, n_pages))


def claim_pages(pages, refs, q_start, context, page, workspace=None):
    """Before a step writes: a page of its own for every block of `page` positions that a sequence's new tokens go to. Missing
    ones come from the free pages (refs under 1), lowest first, and a page that other sequences hold too is replaced.
    pages [b, max_pages] and refs [n_pages] change in place; returns (src, dst, lacking) int32 [b], [b], [1]: copy_pages carries
    src and dst out in every layer's pools, and where lacking is above 0 there were that many free pages too few and nothing was
    changed: the step must wait. The three are parts of one allocation, with up to 1 MB of the call's scratch: a clone keeps less."""
    y = _serving.claim_pages(pages, refs, q_start, context, page, workspace)
    if y is not None:
        return y
    name = "claim_pages"
    b = pages.shape[0] if isinstance(pages, _Tensor) and pages.dim() == 2 else 0
    dev = _table(name, pages, refs, (q_start, "q_start", b + 1), (context, "context", b))
    src, dst, lacking = _empty_i32(b, pages), _empty_i32(b, pages), _empty_i32(1, pages)
    keep, ws, ws_bytes = _bytes(name, dev, workspace, claim_pages_workspace_bytes(b, pages.shape[1], refs.numel()), pages)
    _enqueue("dtts_claim_pages", dev, pages.data_ptr(), refs.data_ptr(), q_start.data_ptr(), context.data_ptr(), src.data_ptr(),
             dst.data_ptr(), lacking.data_ptr(), b, int(page), pages.shape[1], refs.numel(), ws, ws_bytes)
    return src, dst, lacking


def trim_pages(pages, refs, context, page, window, sinks=0):
    """Frees, in place, the pages that tokens from position context[s] on see nothing of under `window` and `sinks`."""
    if _serving.trim_pages(pages, refs, context, page, window, sinks) is not None:
        return
    name = "trim_pages"
    b = pages.shape[0] if isinstance(pages, _Tensor) and pages.dim() == 2 else 0
    dev = _table(name, pages, refs, (context, "context", b))
    _enqueue("dtts_trim_pages", dev, pages.data_ptr(), refs.data_ptr(), context.data_ptr(), b, int(page), pages.shape[1], refs.numel(),
             int(window), int(sinks))


def compact_pages_workspace_bytes(n_pages):
    return int(lib().dtts_compact_pages_workspace_bytes(n_pages))


def compact_pages(pages, refs, workspace=None):
    """Gives the pages in use the first ids, so that a pool can end after them: pages and refs change in place; returns (src, dst,
    used) int32 [n_pages], [n_pages], [1]: the moves that copy_pages carries out in every layer's pools, and how many pages are
    in use. Other tables over the same pools hold none of these ids any more. The three are parts of one allocation, with up to 1 MB
    of the call's scratch: a clone keeps less."""
    y = _serving.compact_pages(pages, refs, workspace)
    if y is not None:
        return y
    name = "compact_pages"
    dev = _table(name, pages, refs)
    n = refs.numel()
    src, dst, used = _empty_i32(n, pages), _empty_i32(n, pages), _empty_i32(1, pages)
    keep, ws, ws_bytes = _bytes(name, dev, workspace, compact_pages_workspace_bytes(n), pages)
    _enqueue("dtts_compact_pages", dev, pages.data_ptr(), refs.data_ptr(), src.data_ptr(), dst.data_ptr(), used.data_ptr(),
             pages.shape[0], pages.shape[1], n, ws, ws_bytes)
    return src, dst, used


def copy_pages(caches, src, dst):
    """Page src[i] to page dst[i] (int32) in each of `caches`, tensors [n_pages, ...] whose pages are contiguous and some
    multiple of 16 bytes: f16 and 4-bit pages of any number of layers at once. Pairs with an id outside the pool (the -1 of
    claim_pages and compact_pages) copy nothing. A page is the destination of one pair at most, and then no source. Two caches share
    no memory, unless they are the same, nor does one with src or dst."""
    if isinstance(caches, _Tensor):
        caches = (caches,)
    if _serving.copy_pages(caches, src, dst) is not None:
        return
    name = "copy_pages"
    if not isinstance(src, _Tensor):
        raise DttsError(f"{name}: src must be a tensor")
    dev = src.get_device()
    _need(name, dev, "src", src, (_I32,))
    _need(name, dev, "dst", dst, (_I32,))
    if src.numel() != dst.numel():
        raise DttsError(f"{name}: {src.numel()} sources and {dst.numel()} destinations")
    caches = list(caches)
    at, size, stride = ((t * len(caches))() for t in (ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64))
    for i, t in enumerate(caches):
        if not isinstance(t, _Tensor):
            raise DttsError(f"{name}: cache {i} must be a tensor")
        _need(name, dev, f"cache {i}", t, (t.dtype,), contiguous=False)
        if t.dim() < 2 or t.shape[0] != caches[0].shape[0] or t.numel() == 0 or not t[0].is_contiguous():
            raise DttsError(f"{name}: cache {i} {tuple(t.shape)} {t.stride()} is not [{caches[0].shape[0]}, ...] with contiguous pages")
        at[i] = t.data_ptr()
        size[i] = t[0].numel() * t.element_size()
        stride[i] = t.stride(0) * t.element_size() if t.shape[0] > 1 else size[i]
    if caches:
        _enqueue("dtts_copy_pages", dev, at, size, stride, len(caches), src.data_ptr(), dst.data_ptr(), src.numel(), caches[0].shape[0])


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
