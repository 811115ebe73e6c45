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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("parts", [0.4, 200.4])
def test_small_slopes_keep_their_digits_over_long_distances(cuda, parts, dtype):
    """Slopes / scale of `parts` 2^-24, subnormal in fp16, and keys some 64,000 places away, the only ones that a mask
    leaves: 0.4 2^-24 of a slope lost would move each probability by 0.4 2^-24 64,000 scale = 2 %, all by as
    much; the bound is u and 65,000 e = 0.4 % (and in bf16 u = 0.4 % itself)."""
    scale, far, heads = 16.0, 64000, 4
    q, k, v, dout = tensors(192, far + 192, heads, 1, 32, dtype, gain=0.05)
    k = (k.float() * 0.05).to(dtype)
    mask = torch.zeros(len(k), dtype=torch.bool, device="cuda")
    mask[:300] = True
    slopes = (scale * parts * 2.0 ** -24 * 0.7 ** torch.arange(heads, dtype=torch.float64)).float().cuda()
    check(q, k, v, [192], [len(k)], dout=dout.abs(), mask=mask, slopes=slopes, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("low", [-65504.0, -1.1e5, -1e9, -1e12, -3e29])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("n,heads", [(440, 32), (300, 2), (48, 2)])
def test_numbers_that_stand_for_not_seen(cuda, n, heads, causal, low, dtype):
    """A window of seven tokens by a bias, and a padded sequence: rows that see no key inside their window. With
    -65504 its keys share such a row, as in a softmax of 32 bits; below -1e5 it is a row without keys."""
    q, k, v, dout = tensors(n, n, heads, heads // 2, 64, dtype, gain=6.0)
    mask = torch.arange(n, device="cuda") < n // 3
    dout[n // 3:] = 0  # nothing is asked of padding
    bias = torch.tensor([[0.0], [low]]).expand(2, heads).cuda()
    buckets = torch.tensor([1, 0, 0, 0, 0, 0, 0, 0, 1], dtype=torch.int32).cuda()
    out, _, grads = check(q, k, v, [n], dout=dout, mask=mask, causal=causal, bias=bias, buckets=buckets)
    if low < -1e5:
        assert not out[n // 3 + 4:].any() and not grads[3][1].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steep", [1e4, 1e6, 3e7, 1e12])
@pytest.mark.parametrize("kind", ["", "cap"])
@pytest.mark.parametrize("n,heads", [(440, 32), (300, 2), (48, 2), (2000, 1)])
def test_rows_far_from_all_keys_they_see(cuda, n, heads, kind, steep, dtype):
    """Steep slopes and a padded sequence, whose last rows see distant keys alone: a cost that fp32 keeps to half a
    power of two is the row's score, one beyond leaves a row without keys."""
    q, k, v, dout = tensors(n, n, heads, max(heads // 4, 1), 64, dtype, gain=6.0)
    mask = torch.arange(n, device="cuda") < n // 3
    dout[n // 3:] = 0  # nothing is asked of padding
    slopes = torch.full((heads,), steep).cuda()
    slopes[1::3] = 0.25
    kw = dict(cap=20.0) if kind else {}
    out, _, _ = check(q, k, v, [n], dout=dout, mask=mask, slopes=slopes, **kw)
    if steep > 2.9e6:
        assert not out[n // 3:, ::3].any()


@pytest.mark.parametrize("steep", [1e4, 3e7])
def test_single_tokens_far_from_all_keys_they_see(cuda, steep):
    from hi3d_amd import attention

    q, k, v, _ = tensors(2, 2 * 9000, 4, 1, 64, torch.float16, gain=6.0)
    mask = (torch.arange(9000, device="cuda") < 5000).expand(2, -1)
    slopes = torch.full((4,), steep).cuda()
    out, lse = attention.attend(q[:, None], k.view(2, 9000, 1, 64), v.view(2, 9000, 1, 64), key_mask=mask, slopes=slopes, return_lse=True)
    shared = attention.attend_shared(q[:, None], k[:4000], v[:4000], k.view(2, 9000, 1, 64)[:, 4000:], v.view(2, 9000, 1, 64)[:, 4000:],
                                     key_mask=mask[:, 4000:], slopes=slopes)
    assert not out.any() and bool(torch.isneginf(lse).all()) and not shared.any()
