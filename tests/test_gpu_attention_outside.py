"""Rows outside the offsets: zeros in outputs and gradients, whatever they and the memory of the
outputs held, and no part in the others' results."""

from __future__ import annotations

import pytest
import torch

from test_gpu_attention import DTYPES, _check_forward, _cu, _tensors
from test_gpu_attention_grad import _check

pytestmark = pytest.mark.gpu


def _poison(*shapes):
    """Leaves NaN in memory that the allocator hands out next."""
    held = [torch.full(shape, float("nan"), device="cuda", dtype=dtype) for shape, dtype in shapes for _ in range(3)]
    torch.cuda.synchronize()
    del held


CASES = [  # lengths of queries and keys, rows in front and behind of queries and of keys
    ([130, 0, 64, 200], None, (0, 77), None),
    ([130, 0, 64, 200], None, (77, 0), None),
    ([130, 0, 64, 200], None, (301, 300), None),
    ([130, 1], [64, 0], (1, 31), (300, 129)),
    ([48] * 100 + [7], None, (50, 400), None),  # a wave to a window
    ([700, 30], [300, 500], (64, 600), (129, 1)),
    ([1] * 70, [500] * 70, (3, 40), (0, 200)),  # single rows, split over the keys
    ([0], [0], (40, 0), (0, 50)),
    ([9], [3000], (0, 60), (5, 5)),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("hq,hk,d", [(3, 3, 64), (4, 1, 88)])
def test_rows_outside_the_offsets(cuda, hq, hk, d, case, causal, dtype):
    from hi3d_amd import attention

    lq, lk, out_q, out_k = CASES[case]
    lk, out_k = lq if lk is None else lk, out_q if out_k is None else out_k
    cu_q, cu_k = _cu(lq) + out_q[0], _cu(lk) + out_k[0]
    nq, nk = int(cu_q[-1]) + out_q[1], int(cu_k[-1]) + out_k[1]
    q, k, v = _tensors(nq, nk, hq, hk, d, dtype, seed=case)
    dout, dlse = _tensors(nq, 1, hq, 1, d, dtype, seed=case + 1)[0], torch.randn(nq, hq, device="cuda")
    in_q, in_k = slice(int(cu_q[0]), int(cu_q[-1])), slice(int(cu_k[0]), int(cu_k[-1]))
    for x, inside in ((q, in_q), (dout, in_q), (dlse, in_q), (k, in_k), (v, in_k)):
        x[:inside.start], x[inside.stop:] = float("nan"), float("nan")
    at = [torch.tensor(x, dtype=torch.int32).cuda() for x in (cu_q, cu_k)]
    _poison((q.shape, dtype), (q.shape[:2], torch.float32))
    out, lse = attention.attend(q, k, v, *at, causal=causal, return_lse=True)
    _check_forward(out[in_q], lse[in_q], q[in_q], k[in_k], v[in_k], cu_q - cu_q[0], cu_k - cu_k[0], causal=causal)
    assert not out[:in_q.start].any() and not out[in_q.stop:].any()
    assert bool(torch.isneginf(lse[:in_q.start]).all()) and bool(torch.isneginf(lse[in_q.stop:]).all())
    _poison((q.shape, dtype), (k.shape, dtype))
    dq, dk, dv = attention.attend_grad(q, k, v, out, lse, dout, *at, dlse=dlse, causal=causal)
    _check((dq[in_q], dk[in_k], dv[in_k]), q[in_q], k[in_k], v[in_k], dout[in_q], cu_q - cu_q[0], cu_k - cu_k[0],
           causal=causal, dlse=dlse[in_q])
    for x, inside in ((dq, in_q), (dk, in_k), (dv, in_k)):
        assert not x[:inside.start].any() and not x[inside.stop:].any()
