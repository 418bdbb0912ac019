"""What dtts.serving checks on the host, beyond the refusals of each call."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from dtts import DttsError, _lib, serving


def test_the_stride_of_a_size_of_one_is_no_ones():
    """contiguous() leaves any number as the stride of a size of 1 (here by transposes): such rows and pages are contiguous."""
    x = torch.zeros((1, 5, 64)).transpose(0, 1)
    assert x.is_contiguous() and x.stride() != (64, 64, 1)
    assert serving._rows("f", x, "x") == ((5, 1, 64), 64)
    assert serving._rows("f", x.transpose(0, 1)[:, :, :].as_strided((1, 5, 64), (3, 64, 1)), "x") == ((1, 5, 64), 320)
    pages = torch.zeros((7, 16, 1, 64)).transpose(1, 2)
    assert serving._page_stride("f", pages) == 1024
    assert serving._page_stride("f", torch.zeros((1, 2, 16, 64)).as_strided((1, 2, 16, 64), (5, 1024, 64, 1))) == 2048
    with pytest.raises(DttsError, match="contiguous rows"):
        serving._rows("f", torch.zeros((2, 5, 64)).transpose(0, 1), "x")
    with pytest.raises(DttsError, match="a page must be contiguous"):
        serving._page_stride("f", torch.zeros((7, 16, 2, 64)).transpose(1, 2))


def _at(n):
    return ctypes.c_void_p(1 << 20 | n)  # an address that no refused call reads


def _refused(fn, match, *args):
    rc = getattr(_lib.lib(), fn)(*args)
    assert rc == -1 and match in _lib.lib().dtts_last_error().decode(), (rc, _lib.lib().dtts_last_error())


@pytest.mark.parametrize("q,q_stride,out", [
    (4096, 512, 4096 + 512), (4096, 512, 4096 + 1536 - 16), (4096, 512, 4096 - 1536 + 16),  # packed queries, from either end
    (0, 4096, 16), (0, 4096, 4096 - 1536 + 16), (0, 4096, 2 * 4096 + 512 - 16),  # in wider rows
])
def test_attention_refuses_an_output_inside_the_queries(q, q_stride, out):
    """Three tokens of 4 heads of 64 (512 bytes a row), an output of 1536 bytes that starts or ends in one of them."""
    p = _at(1 << 16)
    _refused("dtts_paged_attention_f16", "may not be the queries", _at(q), p, p, p, p, p, _at(out), 3, 2, 4, 2, 64, 16, 8, 4, 2048,
             q_stride // 2, 2, 40, 0, 1.0, None, 0, None)


@pytest.mark.parametrize("q_out,k,v,match", [
    (512, 1 << 16, 1 << 17, "may not replace qkv"), (2048 - 16, 1 << 16, 1 << 17, "may not replace qkv"),
    (8192, 1 << 16, 1 << 16, "share memory"), (8192, 1 << 16, (1 << 16) + 4096 - 16, "share memory"),
    (8192, (1 << 16) + 3 * 8192 + 4080, 1 << 16, "share memory"), (8192, 1 << 16, (1 << 16) + 8192 - 16, "share memory"),
])
def test_append_refuses_operands_that_share_memory(q_out, k, v, match):
    """Two f16 tokens of 4 + 2 * 2 heads of 64 (2048 bytes); pages of 4096 bytes, 8192 apart."""
    p = _at(1 << 19)
    _refused("dtts_qk_rope_append_paged_f16", match, _at(0), None, p, p, p, p, p, _at(q_out), _at(k), _at(v), 2, 2, 4, 2, 64, 64, 0,
             16, 8, 4, 4096, 64, 1e-6, None)


@pytest.mark.parametrize("y,ys", [(4, 512), (508, 512), (-508, 512), (1024 + 4, 2048), (-2048, 1024), (3 * 2048, 512)])
def test_rotary_refuses_an_output_partly_inside_x(y, ys):
    """Four f32 rows of 2 heads of 64 (512 bytes), packed or wider, and x or the output in the other's place."""
    p, x = _at(1 << 16), 8192
    xs = 512 if ys != 512 else 2048 if y > 4000 else 512
    _refused("dtts_rotary_f32", "shares memory", _at(x), p, p, p, _at(x + y), 4, 2, 64, 64, 0, xs // 4, ys // 4, 16, None)


def test_the_module_works_without_its_binding():
    """A torch that the binding was not built for: a warning, and every call through Python."""
    code = """
import sys, warnings
sys.modules["dtts._serving"] = None  # an import of it fails
with warnings.catch_warnings(record=True) as met:
    warnings.simplefilter("always")
    from dtts import DttsError, serving
assert len(met) == 1 and "_serving.so" in str(met[0].message), met
import torch
x, i = torch.zeros((2, 2, 64)), torch.zeros(2, dtype=torch.int32)
for call in (lambda: serving.rotary(x, x[0], x[0], i), lambda: serving.sample(x[0], x[0, 0]),
             lambda: serving.paged_attention(x.half(), x, x, i, i, i, 1, 1),
             lambda: serving.qk_rope_append_paged(x[0], x[0], x[0], x, x, i, i, i, 1)):
    try:
        call()
    except DttsError as e:
        assert "on the device" in str(e), e
    else:
        raise AssertionError("taken")
assert serving.rope_table_scaled(4, 8, 1e4)[0].shape == (4, 4)
"""
    subprocess.run([sys.executable, "-c", code], check=True, cwd=os.path.dirname(os.path.dirname(serving.__file__)))
