"""Views with single rows, heads and sequences, whose strides say nothing: the same bits as of
contiguous inputs, forward and gradients."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lead,strides", [
    ((1,), (1347, 64, 1)), ((300,), (64, 3, 1)), ((1,), (1 << 23, 5, 1)), ((1, 1), (999, 1 << 24, 64, 1)),
    ((1, 5), (999, 128, 64, 1)), ((3, 1), (128, 77, 64, 1))])
def test_single_rows_and_heads(cuda, lead, strides):
    from hi3d_amd import attention

    heads = 1 if strides[-2] in (3, 5) else 2
    shape = (*lead, heads, 64)
    room = sum((n - 1) * s for n, s in zip(shape, strides)) + 1
    g = torch.Generator().manual_seed(1)
    plain = [torch.randn(shape, generator=g).half().cuda() for _ in range(4)]
    views = [torch.empty(room, dtype=torch.float16, device="cuda").as_strided(shape, strides) for _ in range(4)]
    for x, y in zip(views, plain):
        x.copy_(y)
    results = []
    for q, k, v, dout in (plain, views):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out, lse = attention.attend(*leaves, return_lse=True)
        assert torch.equal(attention.attend(q, k, v), out)
        results.append([out, lse, *torch.autograd.grad(out, leaves, dout)])
        results[-1] += attention.attend_grad(q, k, v, out.detach(), lse.detach(), dout)
    assert all(torch.equal(a, b) for a, b in zip(*results))
