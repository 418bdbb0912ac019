"""dtts_rotary_{f32,f16} against the rotation in 64 bits: both layouts, part of the head, odd sizes that
take the element kernels, strided rows, in place, padding rows."""
import numpy as np
import pytest
import torch

from dtts import DttsError, ops, serving

import _serving_ref as ref

pytestmark = pytest.mark.gpu


def _case(dev, rows, heads, hd, rot, dtype, seed=0, length=5000):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, heads, hd), generator=g).to(dtype)
    cos, sin = serving.rope_table_scaled(length, rot, 1e4, "yarn", 4.0, length // 4)
    pos = torch.randint(0, length, (rows,), generator=g, dtype=torch.int32)
    return x.to(dev), torch.from_numpy(cos).to(dev), torch.from_numpy(sin).to(dev), pos.to(dev)


def _close(got, x, cos, sin, pos, interleaved):
    p = pos.cpu().numpy()
    want, mag = ref.turn(x.cpu().double().numpy(), cos.cpu().double().numpy()[p], sin.cpu().double().numpy()[p], interleaved)
    # two products and their sum, each rounded to f32; f16 (11 bits, 2^-24 the smallest step) once more
    tol = 2 * 2.0 ** -24 * mag * (1 + 2.0 ** -20)
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -11 * np.abs(want) * (1 + 2.0 ** -10) + 2.0 ** -25
    err = np.abs(got.cpu().double().numpy() - want)
    assert np.all(err <= tol), float(np.max(err - tol))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,hd,rot", [(1, 1, 64, 64), (5, 3, 128, 128), (300, 16, 128, 64), (257, 2, 64, 16), (7, 5, 80, 80),
                                              (9, 2, 128, 6), (3, 2, 40, 12), (2049, 1, 256, 256), (4, 3, 2, 2)])
def test_rotary(dev, rows, heads, hd, rot, interleaved, dtype):
    x, cos, sin, pos = _case(dev, rows, heads, hd, rot, dtype, rows)
    _close(serving.rotary(x, cos, sin, pos, interleaved), x, cos, sin, pos, interleaved)


@pytest.mark.parametrize("hd,rot", [(33, 32), (65, 10), (7, 2)])
def test_rotary_half_split_odd_heads(dev, hd, rot):
    x, cos, sin, pos = _case(dev, 6, 3, hd, rot, torch.float16, hd)
    _close(serving.rotary(x, cos, sin, pos), x, cos, sin, pos, False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rotary_matches_the_host_position_form(dev, dtype):
    x, cos, sin, pos = _case(dev, 100, 4, 128, 128, dtype)
    want = ops.rope(x, cos, sin, pos.cpu().numpy())
    assert torch.equal(serving.rotary(x, cos, sin, pos), want)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [128, 32])
def test_rotary_in_place_on_a_slice_of_qkv(dev, rot, interleaved):
    heads, n_kv, hd, rows = 4, 2, 128, 37
    x, cos, sin, pos = _case(dev, rows, heads + 2 * n_kv, hd, rot, torch.float16, 3)
    before = x.clone()
    k = x[:, heads:heads + n_kv]
    serving.rotary(k, cos, sin, pos, interleaved, out=k)
    _close(x[:, heads:heads + n_kv], before[:, heads:heads + n_kv], cos, sin, pos, interleaved)
    assert torch.equal(x[:, :heads], before[:, :heads]) and torch.equal(x[:, heads + n_kv:], before[:, heads + n_kv:])


def test_rotary_leaves_padding_rows(dev):
    x, cos, sin, pos = _case(dev, 8, 2, 64, 64, torch.float32)
    pos[1], pos[4], pos[7] = -1, cos.shape[0], 2 ** 31 - 1
    out = torch.full_like(x, 7.0)
    serving.rotary(x, cos, sin, pos, out=out)
    pad = [1, 4, 7]
    assert bool((out[pad] == 7.0).all())
    rest = [0, 2, 3, 5, 6]
    _close(out[rest], x[rest], cos, sin, pos[rest], False)


def test_rotary_passes_values_that_are_not_finite_to_their_own_pair_only(dev):
    x, cos, sin, pos = _case(dev, 2, 1, 64, 32, torch.float32)
    x[0, 0, 3], x[1, 0, 40] = float("nan"), float("inf")
    got = serving.rotary(x, cos, sin, pos)
    bad = ~torch.isfinite(got)
    assert bad[0, 0].nonzero().flatten().tolist() == [3, 19] and bad[1, 0].nonzero().flatten().tolist() == [40]


def test_rotary_refuses_shapes(dev):
    x, cos, sin, pos = _case(dev, 4, 2, 64, 64, torch.float32)
    with pytest.raises(DttsError, match="positions for"):
        serving.rotary(x, cos, sin, pos[:3])
    with pytest.raises(DttsError, match="contiguous rows"):
        serving.rotary(x.transpose(0, 1), cos, sin, pos[:2])
    with pytest.raises(DttsError, match="rotated dimensions"):
        serving.rotary(x[..., :32].contiguous(), cos, sin, pos)
    with pytest.raises(DttsError, match="dtype"):
        serving.rotary(x, cos, sin, pos.long())
    with pytest.raises(DttsError, match="out"):
        serving.rotary(x, cos, sin, pos, out=torch.empty_like(x, dtype=torch.float16))
