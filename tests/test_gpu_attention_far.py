"""Rows whose byte offsets, and whose element offsets, pass 32 bits: results that hang on those
rows, and on what else would be read in their place."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
N, HK, D = (1 << 22) + 77, 8, 128  # rows of 2 KB: 2^32 bytes at row 2^21, 2^32 elements at row 2^22
FAR = ((1 << 21) + 5, (1 << 22) + 70)
NEAR = (5, 70, (1 << 21) + 70)  # rows that 32-bit offsets would read for them
SCORE = 20.0
SHARE = (N - 2) / (2 * math.exp(SCORE) + N - 2)
"""What all other keys hold of a row, 0.4 %: an fp32 sum, far key first, may lose that much."""


def _cache(device):
    """Keys of score 0, but for two far ones of score 20; values 0, but for the far keys' and
    large ones at the near places."""
    k, v = (torch.zeros(N, HK, D, dtype=torch.bfloat16, device=device) for _ in range(2))
    g = torch.Generator().manual_seed(0)
    for row in FAR:
        k[row, :, 0] = SCORE
        v[row] = torch.randn(HK, D, generator=g).bfloat16().to(device)
    for row in NEAR:
        v[row] = -64.0
    return k, v


def _parts(v):
    """Probabilities of a far and of another key, and the output of every head, in float64."""
    total = 2 * math.exp(SCORE) + N - 2
    far, other = math.exp(SCORE) / total, 1 / total
    out = far * sum(v[row].double() for row in FAR) + other * sum(v[row].double() for row in NEAR)
    size = far * sum(v[row].double().abs() for row in FAR) + other * sum(v[row].double().abs() for row in NEAR)
    return far, other, out, size


@pytest.mark.parametrize("nq", [1, 40, 200])
def test_far_keys(cuda, nq):
    """One row (split over the keys), rows of one wave, and several waves."""
    from hi3d_amd import attention

    k, v = _cache("cuda")
    q = torch.zeros(nq, HK, D, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1.0
    out, lse = attention.attend(q, k, v, scale=1.0, return_lse=True)
    _, _, want, size = _parts(v)
    # p and the output rounded once; the sum
    room = U * (size + want.abs()) + (SHARE + 2.0 ** -20) * size
    assert bool(((out.double() - want).abs() <= room).all())
    assert float((lse.double() - math.log(2 * math.exp(SCORE) + N - 2)).abs().max()) <= SHARE + 2.0 ** -15


def test_gradients_of_far_keys(cuda):
    from hi3d_amd import attention

    nq = 40
    k, v = _cache("cuda")
    q = torch.zeros(nq, HK, D, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1.0
    dout = torch.randn(nq, HK, D, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    out, lse = attention.attend(q, k, v, scale=1.0, return_lse=True)
    dq, dk, dv = attention.attend_grad(q, k, v, out, lse, dout, scale=1.0)
    p_far, p_other, o, size = _parts(v)
    do = dout.double()
    delta = (do * o).sum(-1)  # [nq, HK]
    delta_off = (do.abs() * (U * (size + o.abs()) + SHARE * size)).sum(-1)
    dq_want, dq_off = 0.0, 0.0
    for row, p in [(r, p_far) for r in FAR] + [(r, p_other) for r in (*NEAR, 1, 1 << 20, N - 1)]:
        ds = p * ((do * v[row].double()).sum(-1) - delta)
        ds_off = (1.1 * U + SHARE) * ds.abs() + p * delta_off
        if p == p_far:
            dq_want, dq_off = dq_want + ds * SCORE, dq_off + ds_off * SCORE
        for got, want, off in ((dv[row], p * do.sum(0), (1.1 * U + SHARE) * p * do.abs().sum(0)),
                               (dk[row][:, 0], ds.sum(0), ds_off.sum(0))):
            assert bool(((got.double() - want).abs() <= off + U * want.abs()).all()), row
        assert not dk[row][:, 1:].any()
    assert bool(((dq[..., 0].double() - dq_want).abs() <= dq_off + U * dq_want.abs()).all())


@pytest.mark.parametrize("causal", [False, True])
def test_rows_far_apart(cuda, causal):
    """Views whose rows lie 8 MB apart, over 9 GB: the same bits as of contiguous copies, with
    gradients; one segment, and segments of which the last lie past 2^32 elements."""
    from hi3d_amd import attention

    rows, heads, d, step = 1100, 2, 64, 1 << 22
    buffer = torch.empty((rows - 1) * step + 3 * heads * d, dtype=torch.bfloat16, device="cuda")
    qkv = buffer.as_strided((rows, 3 * heads, d), (step, d, 1))
    qkv.copy_(torch.randn(rows, 3 * heads, d, generator=torch.Generator().manual_seed(2)).bfloat16())
    dout = torch.randn(rows, heads, d, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    views = [qkv[:, i * heads:(i + 1) * heads] for i in range(3)]
    plain = [x.contiguous() for x in views]
    for lengths in ([rows], [300, 700, 60, 40], [20] * 55):
        at = attention.offsets(lengths)
        results = []
        for x in (views, plain):
            out, lse = attention.attend(*x, at, causal=causal, return_lse=True)
            results.append([out, lse, *attention.attend_grad(*x, out, lse, dout, at, causal=causal)])
        assert all(torch.equal(a, b) for a, b in zip(*results))
    assert (rows - 1) * step > 1 << 32
