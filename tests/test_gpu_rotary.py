"""Rotary positions against float64.

Tolerance: cosine and sine carry up to 2 ulp of fp32 plus the angle's own rounding to fp32
(half a turn: 2^-24 pi), each product and the sum half an ulp more: 8 * 2^-24 of
|first| + |second| covers them; the output adds half a step of its type."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import rotary as orotary

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _check(y, x, positions, freqs, layout, scale=1.0, inverse=False):
    xs = x.detach().double().cpu().numpy()
    want = orotary.rotate(xs, positions.cpu().numpy(), freqs.cpu().numpy(), layout, scale, inverse)
    got = y.detach().double().cpu().numpy()
    reach = np.abs(xs).max(-1, keepdims=True) * 2 * abs(scale)
    tol = HALF_STEP[x.dtype] * np.abs(want) + 8 * 2.0 ** -24 * reach + (2.0 ** -25 if x.dtype == torch.float16 else 0)
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)
    rot = 2 * freqs.shape[1]
    assert np.array_equal(got[..., rot:], xs[..., rot:])


def _inputs(n, hq, hk, dim, axes, rot, dtype, seed=0, far=1000):
    from hi3d_amd import rotary

    g = torch.Generator().manual_seed(seed)
    q, k = torch.randn((n, hq, dim), generator=g).to(dtype).cuda(), torch.randn((n, hk, dim), generator=g).to(dtype).cuda()
    positions = torch.randint(-far, far, (n, axes), generator=g, dtype=torch.int32).cuda()
    return q, k, positions, rotary.frequencies(rot, axes=axes, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("n,hq,hk,dim,rot,axes", [
    (1, 32, 8, 128, 128, 1), (37, 33, 33, 64, 64, 3), (130, 5, 1, 88, 44, 2), (3, 1, 1, 2, 2, 1), (19, 3, 2, 33, 14, 1),
    (65, 4, 4, 96, 0, 1), (8, 2, 2, 1024, 1024, 4), (513, 12, 1, 64, 32, 3)])
def test_forward(cuda, n, hq, hk, dim, rot, axes, layout, dtype):
    from hi3d_amd import rotary

    q, k, positions, freqs = _inputs(n, hq, hk, dim, axes, rot, dtype)
    a, b = rotary.rotate_qk(q, k, positions, freqs, layout=layout, scale=1.25)
    _check(a, q, positions, freqs, layout, 1.25)
    _check(b, k, positions, freqs, layout, 1.25)
    assert torch.equal(rotary.rotate(q, positions, freqs, layout=layout, scale=1.25), a)


def test_far_positions_and_int64(cuda):
    from hi3d_amd import rotary

    q, k, _, freqs = _inputs(64, 4, 2, 64, 1, 64, torch.float32)
    positions = (torch.arange(64, dtype=torch.int64) * 33_333_333 + (1 << 30)).cuda()
    a, b = rotary.rotate_qk(q, k, positions, freqs)
    _check(a, q, positions[:, None], freqs, "half")
    _check(b, k, positions[:, None], freqs, "half")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_views_strides_and_batches(cuda, layout):
    from hi3d_amd import rotary

    _, _, _, freqs = _inputs(1, 1, 1, 64, 3, 64, torch.float16)
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn((77, 11 + 4 + 4, 64), generator=g).half().cuda()
    coords = torch.randint(0, 512, (77, 4), generator=g, dtype=torch.int32).cuda()
    before = qkv.clone()
    a, b = rotary.rotate_qk(qkv[:, :11], qkv[:, 11:15], coords[:, 1:], freqs, layout=layout)
    _check(a, qkv[:, :11], coords[:, 1:], freqs, layout)
    _check(b, qkv[:, 11:15], coords[:, 1:], freqs, layout)
    assert torch.equal(qkv, before)
    # odd row stride and offset: scalar path
    odd = torch.randn((21 * (3 * 64 + 5) + 1,), generator=g).half().cuda()[1:].as_strided((21, 3, 64), (197, 64, 1))
    _check(rotary.rotate(odd, coords[:21, 1:], freqs, layout=layout), odd, coords[:21, 1:], freqs, layout)
    # heads outermost, and a head broadcast to several
    swapped = torch.randn((4, 30, 64), generator=g).half().cuda().transpose(0, 1)
    _check(rotary.rotate(swapped, coords[:30, 1:], freqs, layout=layout), swapped, coords[:30, 1:], freqs, layout)
    wide = torch.randn((30, 1, 64), generator=g).half().cuda().expand(30, 6, 64)
    _check(rotary.rotate(wide, coords[:30, 1:], freqs, layout=layout), wide, coords[:30, 1:], freqs, layout)
    # batches
    x = torch.randn((2, 9, 3, 64), generator=g).half().cuda()
    y = rotary.rotate(x, coords[:18, 1:].reshape(2, 9, 3), freqs, layout=layout)
    assert y.shape == x.shape
    _check(y.reshape(18, 3, 64), x.reshape(18, 3, 64), coords[:18, 1:], freqs, layout)


def test_empty(cuda):
    from hi3d_amd import rotary

    q, k, positions, freqs = _inputs(4, 2, 1, 64, 1, 64, torch.float16)
    a, b = rotary.rotate_qk(q[:0], k[:0], positions[:0], freqs)
    assert a.shape == (0, 2, 64) and b.shape == (0, 1, 64)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_is_the_opposite_rotation(cuda, layout):
    from hi3d_amd import rotary

    q, k, positions, freqs = _inputs(41, 6, 2, 64, 3, 48, torch.float32)
    q.requires_grad_(True)
    base = torch.randn((41, 1, 64), device="cuda", requires_grad=True)  # a broadcast key head
    a, b = rotary.rotate_qk(q, base.expand(41, 2, 64), positions, freqs, layout=layout, scale=0.75)
    da, db = torch.randn_like(a), torch.randn_like(b)
    dq, dk = torch.autograd.grad((a, b), (q, base), (da, db), create_graph=True)
    _check(dq, da, positions, freqs, layout, 0.75, inverse=True)
    each = orotary.rotate(db.double().cpu().numpy(), positions.cpu().numpy(), freqs.cpu().numpy(), layout, 0.75, True)
    got = dk.detach().double().cpu().numpy()
    assert np.abs(got - each.sum(1, keepdims=True)).max() <= 4 * 8 * 2.0 ** -24 * 2 * np.abs(each).max()
    # only one of two outputs used; and against differences along a direction
    assert torch.equal(torch.autograd.grad(rotary.rotate_qk(q, k, positions, freqs, layout=layout, scale=0.75)[0], q, da)[0], dq)
    way = torch.randn_like(q)
    f = lambda x: (rotary.rotate(x, positions, freqs, layout=layout, scale=0.75).double() * da.double()).sum()  # noqa: E731
    with torch.no_grad():  # linear: a difference is exact up to rounding
        step = (f(q + way) - f(q - way)) / 2
    inner = (dq.double() * way.double()).sum()
    room = 16 * 2.0 ** -24 * (da.double().abs() * (q.double().abs() + way.double().abs()).amax(-1, keepdim=True)).sum()
    assert abs(float((step - inner).detach())) <= float(room.detach())


def test_graph_replays(cuda):
    from hi3d_amd import rotary

    q, k, positions, freqs = _inputs(50, 4, 4, 64, 1, 64, torch.float16)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        rotary.rotate_qk(q, k, positions, freqs)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = rotary.rotate_qk(q, k, positions, freqs)
    for i in range(3):
        q.copy_(torch.randn_like(q))
        positions.add_(7 * i)
        graph.replay()
        torch.cuda.synchronize()
        x, y = rotary.rotate_qk(q, k, positions, freqs)
        assert torch.equal(a, x) and torch.equal(b, y)
