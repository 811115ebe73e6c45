"""Attention with terms at the ends of its types' ranges: large and small values behind capped scores, slopes
that 16 bits hold as subnormal numbers, constants that stand for "not seen" in a learned bias."""

from __future__ import annotations

import pytest
import torch

from terms_check import DTYPES, check, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [2.0 ** 100, 2.0 ** -100])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("cap", [3.0, 30.0, 55.0])
def test_values_of_any_size_behind_capped_scores(cuda, cap, d, size):
    """Scores near +cap and -cap, whose exponentials times the values leave fp32 unless they are taken
    relative to the row's largest. (bf16: the values are in its range, and so is the output.)"""
    q, k, v, _ = tensors(440, 440, 32, 8, d, torch.bfloat16)
    at_the_bend = 2.0 * cap * (1.0 + 0.2 * k.float()) / d ** 0.5  # times q of +-1: x = +-2 cap, a row's sign
    sign = torch.where(torch.arange(440, device="cuda")[:, None, None] % 2 == 0, 1.0, -1.0)
    q, k = (sign.expand(q.shape)).to(q.dtype).contiguous(), at_the_bend.to(k.dtype)
    v = (v.float() * size).to(v.dtype)
    check(q, k, v, [220, 220], cap=cap)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("cap", [1e-6, 1e-3, 3.0, 1024.0])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 40, 2.0 ** 55])
def test_large_gradients_of_capped_scores(cuda, size, cap, masked):
    """Pairs that a causal row does not see give nothing, however large dout v is: 2^110 and 64 of them are in
    bf16's range."""
    q, k, v, dout = tensors(440, 440, 32, 8, 64, torch.bfloat16)
    v, dout = ((x.float() * size).to(x.dtype) for x in (v, dout))
    mask = (torch.rand(440, generator=torch.Generator().manual_seed(5)) < 0.7).cuda() if masked else None
    check(q, k, v, [220, 220], dout=dout, causal=True, mask=mask, cap=cap)
