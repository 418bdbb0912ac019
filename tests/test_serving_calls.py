"""What dtts.serving checks on the host, beyond the refusals of each call."""
import pytest
import torch

from dtts import DttsError, serving


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
