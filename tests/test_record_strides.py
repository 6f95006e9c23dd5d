"""Strides that the params records carry in 32 bits (CPU, tensors without memory)."""
import pytest
import torch

import roost_amd


def _meta(shape, strides):
    return torch.empty_strided(shape, strides, device="meta", dtype=torch.bfloat16)


@pytest.mark.parametrize("stride", [2 ** 32, 2 ** 32 + 128, 2 ** 40])
def test_a_stride_of_more_than_32_bits_is_refused(stride):
    """It would be cut to its low bits, and other rows be read."""
    with pytest.raises(ValueError, match="k: tokens are"):
        roost_amd._token_heads(_meta((2, 2, 64), (stride, 64, 1)), "k", 2, 2, 64)
    with pytest.raises(ValueError, match="x: rows are"):
        roost_amd._rows(_meta((2, 128), (stride, 1)), "x", 2, 128)
    # One row has no distance to another.
    assert roost_amd._token_heads(_meta((1, 2, 64), (stride, 64, 1)), "k", 1, 2, 64)[1] == 128
    assert roost_amd._rows(_meta((1, 128), (stride, 1)), "x", 1, 128)[1] == 128


def test_the_largest_stride():
    assert roost_amd._token_heads(_meta((2, 2, 64), (2 ** 32 - 8, 64, 1)), "k", 2, 2, 64)[1] == 2 ** 32 - 8
    for call, shape, strides, args in ((roost_amd._token_heads, (2, 2, 64), (127, 64, 1), (2, 2, 64)),
                                       (roost_amd._rows, (2, 128), (127, 1), (2, 128))):
        with pytest.raises(ValueError, match="127 elements apart, below their 128"):
            call(_meta(shape, strides), "x", *args)
