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


ROWS_33_TO_64 = [
    ([40, 64, 33, 0, 50] * 30, [200, 129, 300, 150, 140] * 30),  # 64 rows to a wave, keys whole
    ([50, 64, 35], [9001, 12000, 8500]),  # and split
]
ROWS_TO_32 = [
    ([20, 32, 1, 0, 9] * 60, [200, 129, 300, 150, 140] * 60),
    ([1, 32, 5], [9001, 12000, 8500]),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("d", [32, 64, 88, 96, 128])
@pytest.mark.parametrize("case", range(4))
def test_one_wave_over_many_keys(cuda, case, d, masked, causal):
    lq, lk = (ROWS_33_TO_64 + ROWS_TO_32)[case]
    mask = (torch.rand(sum(lk), generator=torch.Generator().manual_seed(case)) < 0.7).cuda() if masked else None
    _segments(lq, lk, 2, 2, d, DTYPES[d % 3 == 0], seed=case, causal=causal, mask=mask, grads=False)


@pytest.mark.parametrize("d", [64, 128])
def test_many_heads_on_one_key_head_over_a_cache(cuda, d):
    """64 query heads of one token, and 16 tokens of 4 heads: 64 packed rows over long caches."""
    _segments([1, 1], [9000, 300], 64, 1, d, torch.bfloat16, grads=False)
    _segments([16, 9], [9000, 8000], 8, 2, d, torch.float16, causal=True, grads=False)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk", [
    ([2] * 200 + [3000], None), ([3000] + [0] * 90 + [1] * 150, None), ([5] * 100 + [400], [100] * 100 + [2500]),
    ([30] * 50 + [1], [3] * 50 + [4000])])
def test_segments_far_from_their_average(cuda, lq, lk, causal):
    """The rules go by the average; a segment many times longer is right all the same."""
    _segments(lq, lq if lk is None else lk, 2, 1, 64, torch.float16, causal=causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal,masked", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("nq,cache,hq,hk,d,lens", [
    (9, 150, 4, 2, 64, [150, 0, 1, 77]), (70, 300, 3, 3, 88, [300, 69, 71, 0]), (1, 5000, 8, 2, 128, [5000, 17, 0, 4999]),
    (130, 2000, 2, 1, 32, [2000, 1, 130, 1999]), (50, 9000, 2, 2, 96, [9000, 40, 8999, 64])])
def test_several_rows_over_caches(cuda, nq, cache, hq, hk, d, lens, causal, masked, dtype):
    """Rows end at the last key in use; what lies past those, or is hidden, may hold anything."""
    from hi3d_amd import attention

    batch = len(lens)
    q, k, v = _tensors(batch * nq, batch * cache, hq, hk, d, dtype)
    dout = _tensors(batch * nq, 1, hq, 1, d, dtype, seed=1)[0]
    used = torch.cat([torch.arange(cache) < n for n in lens]).cuda()
    shown = (torch.rand(batch * cache, generator=torch.Generator().manual_seed(2)) < 0.6).cuda() if masked else None
    kk, vv, mask = k[used], v[used], None if shown is None else shown[used]
    hidden = ~used if shown is None else ~used | ~shown
    k[hidden], v[hidden] = float("nan"), float("inf")
    room = lambda x, n: x.reshape(batch, n, *x.shape[1:])  # noqa: E731
    kw = dict(lens_k=torch.tensor(lens, dtype=torch.int32).cuda(), causal=causal,
              key_mask=None if shown is None else room(shown, cache))
    out, lse = attention.attend(room(q, nq), room(k, cache), room(v, cache), return_lse=True, **kw)
    cu_q, cu_k = _cu([nq] * batch), _cu(lens)
    _check_forward(out.flatten(0, 1), lse.flatten(0, 1), q, kk, vv, cu_q, cu_k, causal=causal, mask=mask)
    dq, dk, dv = attention.attend_grad(room(q, nq), room(k, cache), room(v, cache), out, lse, room(dout, nq), **kw)
    dk, dv = dk.flatten(0, 1), dv.flatten(0, 1)
    assert not dk[hidden].any() and not dv[hidden].any()
    _check((dq.flatten(0, 1), dk[used], dv[used]), q, kk, vv, dout, cu_q, cu_k, causal=causal, mask=mask)


@pytest.mark.parametrize("d,masked", [(88, False), (88, True), (128, True), (40, False)])
def test_streamed_caches_with_masks_and_narrow_heads(cuda, d, masked):
    """Caches past 256 MB whose heads do not fill their rows, or whose mask hides single keys and
    whole tiles."""
    from hi3d_amd import attention

    batch, hq, hk = 5, 8, 4
    room = -(-(280 << 20) // (4 * batch * hk * d))
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn((batch, room, hk, d), generator=g, device="cuda").half() for _ in range(2))
    q = torch.randn((batch, 1, hq, d), generator=g, device="cuda").half()
    lens = torch.tensor([room, 17, 0, room - 12, room // 3], dtype=torch.int32, device="cuda")
    mask = torch.rand((batch, room), generator=g, device="cuda") < 0.7
    mask[0, 64 * 20:64 * 90], mask[3, :room // 2], mask[1, :17] = False, False, False
    mask = mask if masked else torch.ones_like(mask)
    k[~mask], v[~mask] = float("nan"), float("nan")
    out = attention.attend(q, k, v, lens_k=lens, key_mask=mask if masked else None)
    assert k.numel() * 4 > 256 << 20
    for b, n in enumerate(lens.tolist()):
        on = mask[b, :n]
        kk, vv = (x[b, :n][on].double().repeat_interleave(hq // hk, 1).transpose(0, 1) for x in (k, v))
        s = (kk * q[b, 0].double()[:, None]).sum(-1) * d ** -0.5
        p = torch.softmax(s, -1) if int(on.sum()) else s
        want, size = (p[..., None] * vv).sum(1), (p[..., None] * vv.abs()).sum(1)
        # p and the output rounded to half a step each; fp32 sums of up to 400,000 terms in parts: 2^-14
        room_ = 2.0 ** -11 * (size + want.abs()) + 2.0 ** -14 * size + 2.0 ** -24
        assert bool(((out[b, 0].double() - want).abs() <= room_).all())
