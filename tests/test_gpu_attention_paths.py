"""Attention's kernels and rules that the other tests do not reach. Bounds as in the small tests."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_attention import DTYPES, _check_forward, _cu, _tensors
from test_gpu_attention_grad import _check, _grads

pytestmark = pytest.mark.gpu


def _segments(lq, lk, hq, hk, d, dtype, seed=0, causal=False, mask=None, grads=True):
    """Forward and gradients of segments against float64."""
    from hi3d_amd import attention

    cu_q, cu_k = _cu(lq), _cu(lk)
    q, k, v = _tensors(int(cu_q[-1]), int(cu_k[-1]), hq, hk, d, dtype, seed=seed)
    at = (attention.offsets(lq), attention.offsets(lk))
    out, lse = attention.attend(q, k, v, *at, causal=causal, key_mask=mask, return_lse=True)
    _check_forward(out, lse, q, k, v, cu_q, cu_k, causal=causal, mask=mask)
    if grads:
        dout = _tensors(int(cu_q[-1]), 1, hq, 1, d, dtype, seed=seed + 1)[0]
        got = _grads(q, k, v, dout, *at, causal=causal, key_mask=mask)
        _check(got, q, k, v, dout, cu_q, cu_k, causal=causal, mask=mask)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 88, 128])
@pytest.mark.parametrize("lq,lk", [
    ([64] * 40, [16] * 40),  # the first 32 rows of every segment see no key
    ([600] + [20] * 40, [50] + [16] * 40),  # a task of 256 rows that sees none
    ([100, 33] * 20, [64, 1] * 20)])
def test_short_segments_whose_first_rows_see_no_key(cuda, lq, lk, d, dtype):
    _segments(lq, lk, 3, 3, d, dtype, causal=True, grads=False)


@pytest.mark.parametrize("bits", [24.6, 25.25, 26.0])
@pytest.mark.parametrize("nq,nk,heads,d", [
    (8192, 100_000, 8, 64),  # 256 rows to a workgroup
    (8192, 100_000, 8, 128),  # 128 rows
    (1, 100_000, 2, 64),  # split over the keys
    (20, 2000, 2, 64),  # eight waves on a block
    (20, 100, 2, 64)])  # a wave on its own
def test_many_keys_far_below_the_first(cuda, nq, nk, heads, d, bits):
    """A key of score s, value 0, before many keys of score 0, value 1: out = n / (e^s + n). In
    fp16 a probability is off by 2^-11 of itself or, below the normal range, by 2^-25 where the
    row's largest is 2^7 or more: 2^-32 of the row's sum a key."""
    from hi3d_amd import attention

    dtype, scale, n = torch.float16, 0.125, nk - 1
    first = float(torch.tensor(bits * 0.6931471805599453).half())  # the score, exact in fp16
    q = torch.zeros(nq, heads, d, dtype=dtype, device="cuda")
    k, v = (torch.zeros(nk, heads, d, dtype=dtype, device="cuda") for _ in range(2))
    q[..., 3], k[0, :, 3], v[1:] = 8.0, first, 1.0
    out, lse = attention.attend(q, k, v, scale=scale, return_lse=True)
    total = math.exp(first) + n
    want = n / total
    pe = 2 * (d + 4) * 2.0 ** -24 * first + (16 + nk) * 2.0 ** -24
    room = (2.0 ** -11 + pe) * want + 2.0 ** -32 * n + 2.0 ** -11 * want + 2.0 ** -24
    assert float((out.double() - want).abs().max()) <= room
    assert float((lse.double() - math.log(total)).abs().max()) <= pe + 4 * 2.0 ** -24 * first + 8 * 2.0 ** -24


def test_fp16_gradients_of_the_largest_values(cuda):
    """The range that fp16 gradients are formed in: values of up to 8189, output gradients all of
    one sign, two keys of probability 1/2 and opposite values, where |ds| is largest: by the
    formulas p (1 - p) 2 sum |dout| max |v|."""
    from hi3d_amd import attention

    for gain in (2.0 ** -10, 1.0, 1.999):  # sum |dout| at both ends of a power of two
        q = torch.randn(40, 1, 64, generator=torch.Generator().manual_seed(0)).half().cuda()
        k, v = torch.zeros(2, 1, 64, dtype=torch.float16, device="cuda"), torch.empty(2, 1, 64, dtype=torch.float16, device="cuda")
        k[0, 0, 0], k[1, 0, 0] = 2.0 ** -10, -2.0 ** -10
        v[0], v[1] = 8188.0, -8188.0
        dout = torch.full((40, 1, 64), gain / 64 * 2.0 ** -8, dtype=torch.float16, device="cuda")
        grads = _grads(q, k, v, dout)
        assert all(bool(x.isfinite().all()) for x in grads)
        _check(grads, q, k, v, dout, [0, 40], [0, 2])
        assert attention.attend(q, k, v).isfinite().all()
