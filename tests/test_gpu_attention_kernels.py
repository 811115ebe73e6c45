"""Every kernel of attention and its gradients at every head width and type, masked and not: one
problem for each tile rule and for keys (or rows) whole and split. Bounds as in the small tests."""

from __future__ import annotations

import pytest
import torch

from test_gpu_attention import DTYPES
from test_gpu_attention_paths import _segments

pytestmark = pytest.mark.gpu

FORWARD = {
    "windows, a wave each": ([48, 0, 33, 64, 48, 7] * 12, [48, 5, 64, 65, 0, 100] * 12),
    "eight waves on a block": ([70, 1], [300, 77]),
    "32 rows": ([20, 32, 1, 0, 9] * 60, [200, 129, 300, 150, 140] * 60),
    "32 rows, split": ([1, 32, 5], [9001, 12000, 8500]),
    "64 rows": ([40, 64, 33, 0, 50] * 30, [200, 129, 300, 150, 140] * 30),
    "64 rows, split": ([50, 64, 35], [9001, 12000, 8500]),
    "128 rows": ([100, 260, 0, 70] * 30, [130, 20, 64, 190] * 30),
    "128 rows, split": ([100, 130, 200], [9001, 12000, 8500]),
    "256 rows": ([22001, 1, 400, 11300], [33, 3, 70, 20]),  # for heads of up to 64
}
GRADIENTS = {
    "rows and keys of a wave": ([15, 0, 9, 16] * 80, [20, 32, 0, 9] * 80),
    "keys of a wave, rows split": ([700, 900], [20, 31]),
    "many rows and keys": ([140, 300], [129, 260]),
    "many keys, rows split": ([2500, 700], [150, 40]),
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("rule", FORWARD)
def test_forward(cuda, rule, d, masked, dtype):
    lq, lk = FORWARD[rule]
    heads = 16 if rule == "256 rows" else 2
    mask = (torch.rand(sum(lk), generator=torch.Generator().manual_seed(d)) < 0.7).cuda() if masked else None
    _segments(lq, lk, heads, heads, d, dtype, causal=(d // 32 + masked) % 2 == 0, mask=mask, grads=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("rule", GRADIENTS)
def test_gradients(cuda, rule, d, masked, dtype):
    lq, lk = GRADIENTS[rule]
    mask = (torch.rand(sum(lk), generator=torch.Generator().manual_seed(d)) < 0.7).cuda() if masked else None
    _segments(lq, lk, 4, 2, d, dtype, causal=(d // 32 + masked) % 2 == 0, mask=mask)
