"""What the calls of 4-bit pages, sinks and page management refuse on the host, through the C ABI, with addresses that no refused
call reads (CPU)."""
import ctypes

import pytest
import torch

from dtts import DttsError, _lib, serving

BIG = 1 << 40


def at(n):
    return ctypes.c_void_p((1 << 44) + n)


def refused(fn, match, *args):
    rc = getattr(_lib.lib(), fn)(*args)
    assert rc == -1 and match in _lib.lib().dtts_last_error().decode(), (rc, _lib.lib().dtts_last_error())


def attention(match, bits=4, q=0, k=BIG, v=2 * BIG, out=3 * BIG, tokens=3, b=2, heads=4, n_kv=2, hd=64, page=16, n_pages=8, max_pages=4,
              stride=1280, q_stride=256, max_q=2, max_context=40, window=0, sinks=0, scale=1.0, ws=None, ws_bytes=0):
    i = at(4 * BIG)
    refused("dtts_paged_attention", match, bits, at(q), at(k), at(v), i, i, i, at(out), tokens, b, heads, n_kv, hd, page, n_pages, max_pages,
            stride, q_stride, max_q, max_context, window, sinks, scale, ws, ws_bytes, None)


@pytest.mark.parametrize("match,bad", [
    ("pages of 8 bits", dict(bits=8)), ("pages of 0 bits", dict(bits=0)), ("head_dim", dict(hd=32)), ("head_dim", dict(hd=96)),
    ("page of 24", dict(page=24)), ("page of 8", dict(page=8)), ("page_stride", dict(stride=1264)), ("page_stride", dict(stride=1288)),
    ("page_stride", dict(stride=1 << 32)), ("page_stride", dict(bits=16, stride=1280)), ("sinks", dict(sinks=-1)),
    ("sinks", dict(sinks=1 << 31)), ("window", dict(window=-1)), ("window", dict(window=1 << 31)), ("heads over", dict(heads=3)),
    ("q_stride", dict(q_stride=255)), ("max_q", dict(max_q=0)), ("max_q", dict(max_context=0)), ("misaligned", dict(k=BIG + 8)),
    ("misaligned", dict(v=2 * BIG + 4)), ("misaligned", dict(q=8)), ("scale", dict(scale=float("inf"))), ("scale", dict(scale=float("nan"))),
    ("may not be the queries", dict(out=512)), ("bad shape", dict(n_pages=0)), ("too many", dict(max_pages=1 << 27)),
    ("too many", dict(tokens=1 << 24)), ("too many rows", dict(tokens=(1 << 24) - 1, heads=256, q_stride=256 * 64, out=BIG * 8)),
])
def test_attention(match, bad):
    attention(match, **bad)


@pytest.mark.parametrize("tokens,match", [(65520, "may not be the queries"), (65521, "too many rows")])
@pytest.mark.parametrize("bits", [16, 4])
def test_attention_of_as_many_tiles_as_a_launch_has(bits, tokens, match):
    """4095 and 4096 tiles of 16 rows of 4096 kv heads, under 2^24 workgroups and not: told by what is refused after that."""
    attention(match, bits=bits, tokens=tokens, b=1, heads=4096, n_kv=4096, stride=4096 * 16 * (64 if bits == 16 else 40), q_stride=4096 * 64,
              max_q=1, out=512)


def test_attention_of_nothing_is_taken():
    p = at(0)
    for tokens, b in ((0, 3), (3, 0)):
        assert _lib.lib().dtts_paged_attention(4, p, p, p, p, p, p, p, tokens, b, 4, 2, 64, 16, 8, 4, 1280, 256, 2, 40, 0, 0, 1.0, None, 0,
                                               None) == 0


def test_workspace_bytes():
    """None where nothing is cut or the sizes are impossible; for f16 pages without sinks what it was; never for less than one state a row."""
    f = _lib.lib().dtts_paged_attention_sinks_workspace_bytes
    assert f(16, 48, 48, 16, 8, 128, 1, 1536, 0, 0) == _lib.lib().dtts_paged_attention_workspace_bytes(48, 48, 16, 8, 128, 1, 1536, 0)
    assert f(4, 1, 1, 16, 8, 128, 1, 300, 0, 0) == 0
    for bad in ((8, 1), (4, 0), (4, -1)):
        assert f(*bad, 48, 16, 8, 128, 1, 1536, 0, 0) == 0
    assert f(4, 48, 48, 16, 8, 128, 1, 1536, 0, -1) == 0
    need = f(4, 48, 48, 16, 8, 128, 1, 1536, 0, 0)
    assert need > 0 and need % (48 * 16 * 132 * 4) == 0
    assert f(4, 5, 5, 32, 4, 128, 1, 65000, 0, 0) <= 64 << 20  # bounded however long the contexts are
    assert f(4, 5, 5, 32, 4, 128, 1, 1 << 30, 0, 0) <= 64 << 20
    assert f(4, 48, 48, 16, 8, 128, 1, 1 << 20, 300, 8) < f(4, 48, 48, 16, 8, 128, 1, 1 << 20, 0, 0)  # a window's keys, not the context's
    assert serving.paged_attention_workspace_bytes(48, 48, 16, 8, 128, 1, 1536, bits=4) == need


def append(match, qkv=0, q_out=BIG, k=2 * BIG, v=3 * BIG, stride=1280, rot=64, page=16, hd=64):
    p = at(4 * BIG)
    refused("dtts_qk_rope_append_paged_q4_f16", match, at(qkv), None, p, p, p, p, p, at(q_out), at(k), at(v), 2, 2, 4, 2, hd, rot, 0, page, 8, 4,
            stride, 64, 1e-6, None)


@pytest.mark.parametrize("match,bad", [
    ("page_stride", dict(stride=1264)), ("page_stride", dict(stride=1296 + 8)), ("misaligned", dict(k=2 * BIG + 8)), ("head_dim", dict(hd=80)),
    ("share memory", dict(v=2 * BIG)), ("share memory", dict(v=2 * BIG + 1264)), ("share memory", dict(v=2 * BIG - 7 * 1280 - 16)),
    ("may not replace qkv", dict(q_out=1024)), ("rotated", dict(rot=68)),
])
def test_append(match, bad):
    append(match, **bad)


def unpack(match, k=0, v=BIG, ko=2 * BIG, vo=3 * BIG, n=8, n_pages=8, ids=None, stride=1280, page=16):
    refused("dtts_unpack_pages_q4", match, at(k), at(v), ids, at(ko), at(vo), n, 2, 64, page, n_pages, stride, None)


@pytest.mark.parametrize("match,bad", [
    ("of 8 pages", dict(n=9)), ("pages", dict(n=-1)), ("misaligned", dict(ko=2 * BIG + 8)), ("share memory", dict(ko=0)),
    ("share memory", dict(vo=2 * BIG + 4080)), ("share memory", dict(vo=7 * 1280)), ("page_stride", dict(stride=1024)),
    ("too many pages", dict(n=(1 << 31) - 1, n_pages=(1 << 31) - 1, ko=BIG * 64, vo=BIG * 128)),
])
def test_unpack(match, bad):
    unpack(match, **bad)


def fork(match, pages=0, refs=BIG, parent=2 * BIG, out=3 * BIG, b=3, n=3, m=4, n_pages=9, ws=4 * BIG, ws_bytes=48):
    refused("dtts_fork_pages", match, at(pages), at(refs), at(parent), at(out), b, n, m, n_pages, at(ws) if ws else None, ws_bytes, None)


@pytest.mark.parametrize("match,bad", [
    ("a table of", dict(b=-1)), ("a table of", dict(n=65537)), ("a table of", dict(m=0)), ("a table of", dict(m=1 << 30)),
    ("a table of", dict(n_pages=0)), ("a table of", dict(n_pages=(1 << 24) + 1)), ("misaligned", dict(refs=BIG + 2)),
    ("no part of it", dict(out=16)), ("no part of it", dict(out=0, n=2)), ("workspace of 48", dict(out=0, ws=None)),
    ("workspace of 48", dict(out=0, ws_bytes=47)), ("share memory", dict(out=0, ws=44)), ("share memory", dict(refs=44)),
    ("share memory", dict(parent=BIG + 32)), ("share memory", dict(parent=3 * BIG + 44)),
])
def test_fork(match, bad):
    fork(match, **bad)


def claim(match, pages=0, refs=BIG, start=2 * BIG, ctx=3 * BIG, src=4 * BIG, dst=5 * BIG, lacking=6 * BIG, b=3, page=16, m=4, n_pages=9,
          ws=7 * BIG, ws_bytes=4 * (12 + 9)):
    assert _lib.lib().dtts_claim_pages_workspace_bytes(3, 4, 9) == 4 * (12 + 9)
    refused("dtts_claim_pages", match, at(pages), at(refs), at(start), at(ctx), at(src), at(dst), at(lacking), b, page, m, n_pages, at(ws),
            ws_bytes, None)


@pytest.mark.parametrize("match,bad", [
    ("a table of", dict(b=65537)), ("positions", dict(page=8)), ("positions", dict(page=48)), ("positions", dict(m=1 << 27)),
    ("workspace", dict(ws_bytes=83)), ("misaligned", dict(src=4 * BIG + 1)), ("share memory", dict(dst=4 * BIG + 8)),
    ("share memory", dict(lacking=5 * BIG + 8)), ("share memory", dict(ctx=BIG)), ("share memory", dict(ws=48 - 4)),
    ("share memory", dict(start=4 * BIG)), ("share memory", dict(refs=44)),
])
def test_claim(match, bad):
    claim(match, **bad)


@pytest.mark.parametrize("b,m,match", [(2047, 1049088, "past an int"), (2047, 1049087, "workspace of")])
def test_claim_of_tables_whose_last_round_passes_an_int(b, m, match):
    """2^31 - 512 entries; and 2^31 - 2559, which is told by what is refused next."""
    claim(match, b=b, m=m, ws_bytes=0)


@pytest.mark.parametrize("match,refs,lacking", [
    ("counts or lacking", None, BIG), ("counts or lacking", 2, BIG), ("counts or lacking", 0, None), ("share memory", 0, 32),
])
def test_claim_without_sequences_needs_its_counts(match, refs, lacking):
    """They are read whatever the batch is; the arrays of sequences are not."""
    p = [None if x is None else at(x) for x in (refs, lacking)]
    refused("dtts_claim_pages", match, None, p[0], None, None, None, None, p[1], 0, 16, 4, 9, None, 0, None)


@pytest.mark.parametrize("match,args", [
    ("window 0", (16, 4, 9, 0, 0)), ("window", (16, 4, 9, 1 << 31, 0)), ("sinks", (16, 4, 9, 5, -1)), ("positions", (17, 4, 9, 5, 0)),
    ("a table of", (16, 0, 9, 5, 0)),
])
def test_trim(match, args):
    refused("dtts_trim_pages", match, at(0), at(BIG), at(2 * BIG), 3, *args, None)


def test_trim_of_shared_memory():
    refused("dtts_trim_pages", "share memory", at(0), at(44), at(2 * BIG), 3, 16, 4, 9, 5, 0, None)
    refused("dtts_trim_pages", "share memory", at(0), at(BIG), at(BIG + 32), 3, 16, 4, 9, 5, 0, None)


@pytest.mark.parametrize("match,bad", [
    ("a table of", dict(n_pages=0)), ("workspace", dict(ws_bytes=4 * 9)), ("share memory", dict(dst=2 * BIG + 32)),
    ("share memory", dict(used=BIG)), ("share memory", dict(ws=44)), ("misaligned", dict(used=4 * BIG + 2)),
])
def test_compact(match, bad):
    a = dict(pages=0, refs=BIG, src=2 * BIG, dst=3 * BIG, used=4 * BIG, b=3, m=4, n_pages=9, ws=5 * BIG, ws_bytes=4 * 11) | bad
    assert _lib.lib().dtts_compact_pages_workspace_bytes(9) == 4 * 11
    refused("dtts_compact_pages", match, *(at(a[x]) for x in ("pages", "refs", "src", "dst", "used")), a["b"], a["m"], a["n_pages"],
            at(a["ws"]), a["ws_bytes"], None)


@pytest.mark.parametrize("match,bad", [
    ("multiples of 16", dict(size=24)), ("multiples of 16", dict(stride=1288)), ("multiples of 16", dict(stride=1264)),
    ("multiples of 16", dict(size=0)), ("multiples of 16", dict(size=1 << 29, stride=1 << 29)), ("16-byte aligned", dict(cache=8)),
    ("16-byte aligned", dict(cache=None)), ("pairs in", dict(n=-1)), ("pairs in", dict(n=1 << 31)), ("pairs in", dict(n_caches=65537)),
    ("pairs in", dict(n_pages=0)), ("misaligned", dict(src=BIG + 2)),
])
def test_copy(match, bad):
    a = dict(cache=0, size=1280, stride=1280, n=5, n_pages=9, n_caches=1, src=BIG) | bad
    caches = (ctypes.c_void_p * 1)(None if a["cache"] is None else at(a["cache"]).value)
    refused("dtts_copy_pages", match, caches, (ctypes.c_int64 * 1)(a["size"]), (ctypes.c_int64 * 1)(a["stride"]), a["n_caches"], at(a["src"]),
            at(2 * BIG), a["n"], a["n_pages"], None)


@pytest.mark.parametrize("size", [(1 << 29) - 8192 + 16, (1 << 29) - 16])
def test_copy_of_pages_with_more_slices_than_a_grid_has_rows(size):
    c = (ctypes.c_void_p * 2)(at(0).value, at(BIG).value)
    refused("dtts_copy_pages", "apart", c, (ctypes.c_int64 * 2)(1280, size), (ctypes.c_int64 * 2)(1280, 1 << 30), 2, at(2 * BIG),
            at(3 * BIG), 5, 9, None)


def copy_of(match, *pools, src=8 * BIG, dst=9 * BIG, n=5, n_pages=9):
    """Pools (address, bytes of a page, bytes from page to page)."""
    addresses, sizes, strides = zip(*pools)
    caches = (ctypes.c_void_p * len(pools))(*(at(a).value for a in addresses))
    refused("dtts_copy_pages", match, caches, *((ctypes.c_int64 * len(pools))(*x) for x in (sizes, strides)), len(pools), at(src), at(dst),
            n, n_pages, None)


ONE = (BIG, 1280, 2560)


@pytest.mark.parametrize("match,pools,pairs", [
    ("pairs share memory", [ONE], dict(src=BIG)), ("pairs share memory", [ONE], dict(dst=BIG + 8 * 2560 + 1276)),
    ("pairs share memory", [ONE], dict(src=BIG - 16)), ("pairs share memory", [(0, 64, 64), ONE], dict(dst=BIG + 2560 - 4)),
    ("share memory", [ONE, (BIG + 16, 1280, 2560)], {}), ("share memory", [(BIG + 1264, 1280, 2560), ONE], {}),
    ("share memory", [ONE, (BIG + 1280 + 16, 1280, 2560)], {}), ("share memory", [ONE, (BIG, 1264, 2560)], {}),
    ("share memory", [ONE, (BIG, 1280, 1280)], {}), ("share memory", [ONE, (BIG + 1280, 1280, 1280)], {}),
    ("share memory", [ONE, (BIG - 8 * 2560 - 1264, 1280, 2560)], {}), ("share memory", [ONE, (BIG + 8 * 2560 + 1264, 16, 16)], {}),
    ("share memory", [(BIG + 1280, 1280, 2560), (3 * BIG, 64, 64), ONE, (2 * BIG, 64, 80), (BIG + 1264, 16, 2560)], {}),
])
def test_copy_of_shared_memory(match, pools, pairs):
    copy_of(match, *pools, **pairs)


@pytest.mark.parametrize("pools,pairs", [
    ([ONE, ONE], {}), ([ONE, (BIG + 1280, 1280, 2560)], {}), ([ONE, (BIG + 8 * 2560 + 1280, 64, 64)], {}), ([(BIG - 9 * 64, 64, 64), ONE], {}),
    ([ONE], dict(src=BIG + 1280)), ([ONE], dict(src=BIG + 8 * 2560 + 1280, dst=BIG - 20)),
    ([(BIG + 80 * i, 80, 80 * 64) for i in reversed(range(64))], {}), ([(BIG + 640, 640, 1280), (BIG, 320, 640)], dict(n_pages=1)),
])
def test_copy_of_pools_that_lie_apart(pools, pairs):
    """Told by what is refused after them: two pools past all others."""
    n = len(pools)
    copy_of(f"caches {n} and {n + 1} share memory", *pools, (7 * BIG, 64, 64), (7 * BIG + 32, 64, 64), **pairs)


def test_tensors_that_are_not_on_a_gpu():
    i, x = torch.zeros((2, 2), dtype=torch.int32), torch.zeros((4, 2, 16, 40), dtype=torch.uint8)
    for call in (lambda: serving.fork_pages(i, i[0], i[0]), lambda: serving.claim_pages(i, i[0], torch.zeros(3, dtype=torch.int32), i[0], 16),
                 lambda: serving.trim_pages(i, i[0], i[0], 16, 4), lambda: serving.compact_pages(i, i[0]),
                 lambda: serving.copy_pages([x], i[0], i[0]), lambda: serving.copy_pages(x, i[0], i[0]), lambda: serving.unpack_pages(x, x),
                 lambda: serving.paged_attention(torch.zeros((1, 4, 64), dtype=torch.float16), x, x, i[0], i[0, :1], i[:1], 1, 1, sinks=2)):
        with pytest.raises(DttsError, match="on the device"):
            call()
    for call in (lambda: serving.fork_pages(None, i[0], i[0]), lambda: serving.claim_pages([1], i[0], i[0], i[0], 16),
                 lambda: serving.trim_pages(3, i[0], i[0], 16, 4), lambda: serving.compact_pages("x", i[0]),
                 lambda: serving.copy_pages([x], None, i[0]), lambda: serving.unpack_pages(None, x)):
        with pytest.raises(DttsError, match="must be a tensor"):
            call()


def test_the_binding_takes_no_wrong_call():
    b, i, x = serving._serving, torch.zeros((2, 2), dtype=torch.int32), torch.zeros((4, 2, 16, 40), dtype=torch.uint8)
    assert b.unpack_pages(x, x, None) is None and b.unpack_pages(None, 1, "2") is None
    assert b.fork_pages(i, i[0], i[0], None, None) is None and b.fork_pages(None, 1, 2, 3, 4) is None
    assert b.claim_pages(i, i[0], i[0], i[0], 16, None) is None and b.claim_pages(1, 2, 3, 4, "16", 5) is None
    assert b.trim_pages(i, i[0], i[0], 16, 4, 0) is None and b.compact_pages(i, i[0], None) is None
    assert b.copy_pages([x], i[0], i[0]) is None and b.copy_pages(None, None, None) is None and b.copy_pages([1, 2], i, i) is None
    with pytest.raises(TypeError):
        b.fork_pages(i)
