"""Strides that the attention kernels are given, on the CPU."""

from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("shape,strides", [
    ((1, 7, 64), (1347, 64, 1)),  # one token of rows of an odd width
    ((300, 1, 64), (64, 3, 1)),  # one head
    ((1, 1, 64), (1 << 23, 5, 1)),  # one token of one head, rows far apart
    ((1, 1, 7, 64), (999, 1 << 24, 64, 1)),  # one token of one sequence
    ((1, 5, 2, 64), (999, 128, 64, 1)),
    ((3, 1, 2, 64), (128, 77, 64, 1)),
])
def test_places_of_single_rows_and_heads(shape, strides):
    """The stride of a dimension of one is never used: such a view is read in place, by strides
    that the C entries take (multiples of 8, rows nearer than 2^23)."""
    from hi3d_amd import attention

    room = sum((n - 1) * s for n, s in zip(shape, strides)) + 1
    x = torch.zeros(room, dtype=torch.float16).as_strided(shape, strides)
    y, got = attention._heads(x)
    assert y.data_ptr() == x.data_ptr() and y.shape == x.shape
    assert all(s % 8 == 0 for s in got[:-1]) and 0 <= got[-3] < 1 << 23
    assert all(a == b for a, b, n in zip(got, strides, shape) if n > 1)
