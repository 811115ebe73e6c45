"""Attention's kernels and rules that the other tests do not reach. Bounds as in the small tests."""

from __future__ import annotations

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
