"""Gradients of a learned bias where workgroups' rows see no key: what they leave has to be zeros, whatever
the workgroups before them left in LDS."""

from __future__ import annotations

import pytest
import torch

from terms_check import DTYPES, tensors, terms

pytestmark = pytest.mark.gpu

ROWS, KEYS = 30000, 300  # some 240 workgroups a head without a key


def _problem(case):
    """Lengths, causal or not, and mask of problems none of whose rows sees a key."""
    from hi3d_amd import attention

    mask = None
    if case == "no keys":
        return 0, None, False, mask
    if case == "segments without keys":
        return KEYS, (attention.offsets([10000, 0, 20000, 0]), attention.offsets([0, KEYS, 0, 0])), False, mask
    if case == "rows outside the offsets":
        cu = torch.tensor([500, 500, 500], dtype=torch.int32).cuda()
        return KEYS, (cu, torch.tensor([0, KEYS, KEYS], dtype=torch.int32).cuda()), False, mask
    if case == "rows in front of all keys":  # the last 300 would see some: hidden ones
        mask = torch.zeros(KEYS, dtype=torch.bool).cuda()
    return KEYS, None, True, mask


@pytest.mark.parametrize("case", ["no keys", "segments without keys", "rows outside the offsets", "rows in front of all keys"])
@pytest.mark.parametrize("kind", ["bias", "cap slopes bias"])
@pytest.mark.parametrize("d", [64, 88, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_keys_leave_the_bias_alone(cuda, dtype, d, kind, case):
    from hi3d_amd import attention

    nk, cu, causal, mask = _problem(case)
    q, k, v, dout = tensors(ROWS, nk, 2, 2, d, dtype)
    kw = terms(kind, 2, far=1024, count=64)
    full, _, _, other = tensors(4000, 4000, 2, 2, d, dtype, seed=1)  # leaves its sums and tables in LDS
    for _ in range(2):
        leaves = [x.detach().requires_grad_(True) for x in (full, full, full, kw["bias"])]
        out = attention.attend(*leaves[:3], **dict(kw, bias=leaves[3]))
        assert torch.autograd.grad(out, leaves, other)[3].any()
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v, kw["bias"])]
        out = attention.attend(*leaves[:3], *(cu or ()), causal=causal, key_mask=mask, **dict(kw, bias=leaves[3]))
        grads = torch.autograd.grad(out, leaves, dout)
        assert not out.any() and not any(g.any() for g in grads)


@pytest.mark.parametrize("wanted", ["all", "bias"])
def test_rows_without_keys_beside_rows_with_some(cuda, wanted):
    """The gradient of segments that see keys, with and without 30,000 rows that see none around them: sums in another
    order, within the rounding of sums of some 10^5 numbers in runs of 64 (2^-24 of their magnitude a step, 300
    steps)."""
    from hi3d_amd import attention

    q, k, v, dout = tensors(ROWS + 400, 400, 2, 2, 64, torch.float16)
    kw = terms("bias", 2, far=40)

    def grad(q, k, v, dout, *cu):
        bias = kw["bias"].detach().requires_grad_(True)
        leaves = [x.detach().requires_grad_(wanted == "all") for x in (q, k, v)]
        out = attention.attend(*leaves, *cu, **dict(kw, bias=bias))
        return torch.autograd.grad(out, bias, dout)[0]

    inner = slice(10000, 10400)
    got = grad(q, k, v, dout, attention.offsets([10000, 400, 20000]), attention.offsets([0, 400, 0]))
    want = grad(q[inner], k, v, dout[inner])
    size = (dout[inner].float().abs().sum(-1) * 2 * v.abs().max()).sum()  # of |ds| over a row: sum p = 1
    assert want.any() and bool(((got - want).abs() <= 300 * 2.0 ** -24 * size).all())
