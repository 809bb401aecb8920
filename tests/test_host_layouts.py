"""Outputs that are laid out like an input, without a GPU."""

import itertools

import torch

from cab_attention import _native as nat


def test_rows_of_an_output_are_contiguous():
    """Every shape and stride of small views with a contiguous last dim: the output's is, and its rows lie apart."""
    memory = torch.empty(4096)
    for shape in itertools.product((1, 2), (1, 3), (1, 5), (2, 8)):
        for strides in itertools.product((0, 1, 8, 40), (0, 1, 8, 24), (0, 1, 2, 8)):
            x = memory.as_strided(shape, (*strides, 1))
            y = nat.empty_rows_like(x)
            assert y.shape == x.shape and y.stride(3) == 1
            if torch.empty_like(x).stride(3) == 1:
                assert y.stride() == torch.empty_like(x).stride()
            places = torch.arange(4096).as_strided(y.shape, y.stride()).flatten()
            assert places.unique().numel() == places.numel()
