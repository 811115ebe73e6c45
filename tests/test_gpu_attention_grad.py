"""Gradients of attention against float64 and against differences.

Tolerances follow the roundings, with u half a step of the type and e = 2^-24:

* p is formed again as exp(score - lse): a relative error ``pe`` of the score's (d + 4) e
  ``reach``, of lse's own (as the forward's bound), of lse times log2(e) (2 e |lse|) and 8 e;
* p and ds are rounded to the type: u each, and in fp16 absolute floors: p is scaled by 2^10
  (2^-35 of its own), ds so that 8 or more stands for the largest sum |dout| (2^-28 of that);
* D = sum(dout out) is off by the output's own rounding (the forward's bound) and d e more;
* ``oracle.attention.backward`` carries these through the sums in magnitudes; fp32 sums over n
  rows add n / 16 e of the same magnitudes at most (16 rows to a matrix instruction, whose sums
  are fp32's);
* the gradient is rounded once; products of two relative errors are below 1 %."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import attention as oattention

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
E = 2.0 ** -24
DTYPES = [torch.float16, torch.bfloat16]


def _np(x):
    return None if x is None else x.detach().double().cpu().numpy()


def _cu(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)


def _tensors(nq, nk, hq, hk, d, dtype, seed=0, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    make = lambda n, h, s: (s * torch.randn((n, h, d), generator=g)).to(dtype).cuda()  # noqa: E731
    return make(nq, hq, 1.0), make(nk, hk, 1.0), make(nk, hk, 1.0), make(nq, hq, gain)


def _check(grads, q, k, v, dout, cu_q, cu_k, scale=None, causal=False, mask=None, dlse=None):
    dtype, d = q.dtype, q.shape[-1]
    sq, sk = oattention.spans(cu_q), oattention.spans(cu_k)
    mask = None if mask is None else mask.cpu().numpy()
    f = oattention.forward(_np(q), _np(k), _np(v), sq, sk, scale, causal, mask)
    keys, rows = max([b - a for a, b in sk] + [0]), max([b - a for a, b in sq] + [0]) * (q.shape[1] // k.shape[1])
    p_forward = 2 * (d + 4) * E * f["reach"] + (16 + keys) * E
    lse = np.abs(np.where(np.isneginf(f["lse"]), 0, f["lse"]))
    pe = (d + 4) * E * f["reach"] + p_forward + (4 + 2 + 8) * E * (1 + lse)
    out_off = (U[dtype] + p_forward[..., None]) * f["size"] + TINY[dtype] * f["vsum"] + U[dtype] * np.abs(f["out"]) + 2 * TINY[dtype]
    do = np.abs(_np(dout))
    delta_off = (do * out_off).sum(-1) + (d + 1) * E * (do * np.abs(f["out"])).sum(-1)
    floor = 0.0
    if dtype == torch.float16:
        most = do.sum(-1).max(initial=0)
        if dlse is not None:
            most = max(most, np.abs(_np(dlse)).max(initial=0))
        floor = 2.0 ** -35 + 2.0 ** -28 * most  # of p and of ds: both take the larger
    r = oattention.backward(_np(q), _np(k), _np(v), _np(dout), sq, sk, scale, causal, mask, delta_error=delta_off,
                            p_error=pe + (keys + rows) / 16 * E, u=U[dtype] + 4 * E, floor=floor, dlse=_np(dlse))
    for got, name in zip(grads, ("dq", "dk", "dv")):
        if got is None:
            continue
        assert got.dtype == dtype
        got, want = _np(got), r[name]
        assert np.isfinite(got).all(), f"{name} is not finite"
        room = 1.01 * r[name + "_off"] + U[dtype] * np.abs(want) + 2 * TINY[dtype]
        off = np.abs(got - want)
        assert (off <= room).all(), f"{name}: {np.max(off / np.maximum(room, 1e-300))} of the room"


def _grads(q, k, v, dout, *cu, **kw):
    from hi3d_amd import attention

    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = attention.attend(*leaves, *cu, **kw)
    return torch.autograd.grad(out, leaves, dout)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [8, 32, 40, 64, 88, 96, 120, 128])
def test_head_sizes(cuda, d, dtype):
    q, k, v, dout = _tensors(150, 211, 4, 2, d, dtype)
    _check(_grads(q, k, v, dout), q, k, v, dout, [0, 150], [0, 211])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 2), (2, 1), (31, 33), (32, 32), (63, 65), (64, 64), (65, 63), (127, 129),
                                   (128, 128), (257, 255), (300, 5), (5, 300), (1, 1000), (1000, 1), (517, 517)])
def test_lengths(cuda, nq, nk, causal, dtype):
    q, k, v, dout = _tensors(nq, nk, 2, 2, 64, dtype)
    grads = _grads(q, k, v, dout, causal=causal)
    _check(grads, q, k, v, dout, [0, nq], [0, nk], causal=causal)
    if causal and nq > nk:
        assert not grads[0][:nq - nk].any()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 4), (6, 2), (5, 1), (32, 8), (33, 33)])
def test_grouped_heads(cuda, hq, hk, causal):
    """The query heads of a shared key head sum into its gradients."""
    q, k, v, dout = _tensors(143, 143, hq, hk, 64, torch.bfloat16)
    _check(_grads(q, k, v, dout, causal=causal), q, k, v, dout, [0, 143], [0, 143], causal=causal)


RAGGED = [
    ([48] * 9 + [29], None),
    ([1, 0, 2, 700, 0, 0, 33, 64, 128, 1], None),
    ([0, 0, 5], [0, 7, 0]),
    ([300, 20, 0, 77], [3, 0, 90, 400]),
    ([17] * 200, None),
    ([(7 * i) % 90 for i in range(150)], [(11 * i) % 70 for i in range(150)]),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", range(len(RAGGED)))
@pytest.mark.parametrize("dtype", DTYPES)
def test_segments(cuda, case, causal, dtype):
    from hi3d_amd import attention

    lq, lk = RAGGED[case]
    cu_q, cu_k = _cu(lq), _cu(lk if lk is not None else lq)
    q, k, v, dout = _tensors(int(cu_q[-1]), int(cu_k[-1]), 4, 2, 32, dtype, seed=case)
    kw = {} if lk is None else {"cu_k": attention.offsets(lk)}
    _check(_grads(q, k, v, dout, attention.offsets(lq), causal=causal, **kw), q, k, v, dout, cu_q, cu_k, causal=causal)


@pytest.mark.parametrize("nq,nk,hq,hk", [(3000, 150, 4, 1), (2500, 70, 2, 2), (700, 40, 16, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_few_keys_split_over_the_rows(cuda, nq, nk, hq, hk, causal):
    q, k, v, dout = _tensors(nq, nk, hq, hk, 64, torch.bfloat16)
    _check(_grads(q, k, v, dout, causal=causal), q, k, v, dout, [0, nq], [0, nk], causal=causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), 65504.0])
@pytest.mark.parametrize("d", [64, 88])
def test_hidden_keys_may_hold_anything(cuda, d, fill, dtype):
    from hi3d_amd import attention

    lengths = [130, 64, 1, 200]
    cu = _cu(lengths)
    n = int(cu[-1])
    q, k, v, dout = _tensors(n, n, 3, 3, d, dtype)
    mask = torch.rand(n, generator=torch.Generator().manual_seed(5)) < 0.6
    mask[130:194] = False  # a segment without keys
    mask[64:128] = False  # a whole tile of a segment
    mask = mask.cuda()
    clean = _grads(q, k, v, dout, attention.offsets(lengths), key_mask=mask)
    _check(clean, q, k, v, dout, cu, cu, mask=mask)
    assert not clean[0][130:194].any() and not clean[1][~mask].any() and not clean[2][~mask].any()
    k[~mask], v[~mask] = fill, fill
    for a, b in zip(clean, _grads(q, k, v, dout, attention.offsets(lengths), key_mask=mask)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("gain", [2.0 ** -14, 1.0, 64.0])
def test_fp16_gradients_of_any_size(cuda, gain):
    """Gradients far below 1 over many keys: score gradients near 2^-14 * 2^-11 * dout. And rows
    of very different sizes."""
    q, k, v, dout = _tensors(200, 2048, 2, 2, 64, torch.float16, gain=gain)
    _check(_grads(q, k, v, dout), q, k, v, dout, [0, 200], [0, 2048])
    q, k, v, dout = _tensors(2048, 100, 2, 2, 64, torch.float16, gain=gain)
    dout[::2] *= 2.0 ** -6
    _check(_grads(q, k, v, dout, causal=True), q, k, v, dout, [0, 2048], [0, 100], causal=True)
    zero = _grads(q, k, v, torch.zeros_like(dout))
    assert not any(x.any() for x in zero)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cache_lengths(cuda, dtype):
    """Keys past those in use: never read, and zero gradients."""
    from hi3d_amd import attention

    batch, nq, cache, hq, hk, d, lens = 4, 9, 150, 4, 2, 64, [150, 0, 1, 77]
    q, k, v, dout = _tensors(batch * nq, batch * cache, hq, hk, d, dtype)
    used = torch.cat([torch.arange(cache) < n for n in lens]).cuda()
    keep = [x[used] for x in (k, v)]
    k[~used], v[~used] = float("nan"), float("nan")
    shape = lambda x, n: x.reshape(batch, n, x.shape[1], d)  # noqa: E731
    lens_k = torch.tensor(lens, dtype=torch.int32).cuda()
    dq, dk, dv = _grads(shape(q, nq), shape(k, cache), shape(v, cache), shape(dout, nq), lens_k=lens_k)
    dk, dv = dk.reshape(-1, hk, d), dv.reshape(-1, hk, d)
    assert not dk[~used].any() and not dv[~used].any()
    _check((dq.reshape(-1, hq, d), dk[used], dv[used]), q, *keep, dout, _cu([nq] * batch), _cu(lens))
    assert attention.attend(shape(q, nq), shape(k, cache), shape(v, cache), lens_k=lens_k).isfinite().all()


def test_views_broadcasts_and_parts(cuda):
    """Strided inputs, an output gradient that is a broadcast, a broadcast key head, gradients
    of only some inputs, and of lse."""
    from hi3d_amd import attention

    g = torch.Generator().manual_seed(2)
    qkv = torch.randn((333, 7 + 7 + 7, 64), generator=g).half().cuda().requires_grad_(True)
    dout = torch.randn((333, 7, 64), generator=g).half().cuda()
    out = attention.attend(qkv[:, :7], qkv[:, 7:14], qkv[:, 14:])
    whole, = torch.autograd.grad(out, qkv, dout)
    parts = [qkv.detach()[:, 7 * i:7 * i + 7].contiguous() for i in range(3)]
    want = _grads(*parts, dout)
    for i in range(3):
        assert torch.equal(whole[:, 7 * i:7 * i + 7], want[i])
    row = torch.randn((333, 1, 64), generator=g).half().cuda()
    assert all(torch.equal(a, b) for a, b in zip(_grads(*parts, row.expand(333, 7, 64)),
                                                 _grads(*parts, row.expand(333, 7, 64).contiguous())))
    one = torch.randn((333, 1, 64), generator=g).half().cuda().requires_grad_(True)
    spread, = torch.autograd.grad(attention.attend(parts[0], one.expand(333, 7, 64), parts[2]), one, dout)
    each = _grads(parts[0], one.detach().expand(333, 7, 64), parts[2], dout)[1]
    # torch sums the seven heads itself, in fp32, and rounds once
    exact = each.double().sum(1, keepdim=True)
    assert bool(((spread.double() - exact).abs() <= 2.0 ** -11 * exact.abs() + 7 * E * each.double().abs().sum(1, keepdim=True)
                 + 2.0 ** -25).all())
    for some in ((True, False, False), (False, True, False), (False, False, True)):
        leaves = [x.detach().requires_grad_(on) for x, on in zip(parts, some)]
        got = torch.autograd.grad(attention.attend(*leaves), [x for x, on in zip(leaves, some) if on], dout)
        assert torch.equal(got[0], want[some.index(True)])
    leaves = [x.detach().requires_grad_(True) for x in parts]
    out, lse = attention.attend(*leaves, return_lse=True)
    dlse = torch.randn(lse.shape, generator=g).cuda()
    got = torch.autograd.grad((out, lse), leaves, (dout, dlse))
    _check(got, *parts, dout, [0, 333], [0, 333], dlse=dlse)
    for a, b in zip(got, attention.attend_grad(*parts, out.detach(), lse.detach(), dout, dlse=dlse)):
        assert torch.equal(a, b)
    out, lse = attention.attend(*leaves, return_lse=True)
    only, zero = torch.autograd.grad(lse, leaves, dlse, allow_unused=True), torch.zeros_like(dout)
    _check(only, *parts, zero, [0, 333], [0, 333], dlse=dlse)
    with pytest.raises(RuntimeError):
        first, = torch.autograd.grad(attention.attend(*leaves).float().sum(), leaves[0], create_graph=True)
        first.float().sum().backward()


@pytest.mark.parametrize("causal", [False, True])
def test_against_differences(cuda, causal):
    """<gradient, way> against the loss's central difference along the way, whose forward passes
    are float64: only the gradient's own roundings remain."""
    q, k, v, dout = _tensors(90, 120, 4, 2, 64, torch.bfloat16, seed=3)
    grads = [_np(x) for x in _grads(q, k, v, dout, causal=causal)]
    q, k, v, do = (_np(x) for x in (q, k, v, dout))
    rng = np.random.default_rng(4)
    for i in range(3):
        way = rng.standard_normal((q, k, v)[i].shape)
        step = 1e-5
        losses = []
        for s in (step, -step):
            x = [q, k, v]
            x[i] = x[i] + s * way
            losses.append((oattention.forward(*x, [(0, 90)], [(0, 120)], None, causal)["out"] * do).sum())
        slope = (losses[0] - losses[1]) / (2 * step)
        inner = (grads[i] * way).sum()
        # the gradient's elements carry about two roundings (2^-8 each) with random signs
        room = 6 * 2.0 ** -7 * np.sqrt((grads[i] ** 2 * way ** 2).sum())
        assert abs(slope - inner) <= room, (slope, inner, room)


def test_empty(cuda):
    from hi3d_amd import attention

    q, k, v, dout = _tensors(10, 12, 2, 2, 64, torch.float16)
    dq, dk, dv = _grads(q[:0], k, v, dout[:0])
    assert dq.shape == (0, 2, 64) and not dk.any() and not dv.any()
    dq, dk, dv = _grads(q, k[:0], v[:0], dout)
    assert not dq.any() and dk.shape == (0, 2, 64)
    assert [x.shape[0] for x in _grads(q[:0], k[:0], v[:0], dout[:0], attention.offsets([]))] == [0, 0, 0]
    dq, dk, dv = _grads(q, k, v, dout, attention.offsets([10, 0]), attention.offsets([0, 12]))
    assert not dq.any() and not dk.any() and not dv.any()


def test_same_bits_every_time_and_on_another_stream(cuda):
    q, k, v, dout = _tensors(2000, 200, 8, 1, 128, torch.bfloat16)
    want = _grads(q, k, v, dout)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(_grads(q, k, v, dout), want))
    torch.cuda.current_stream().wait_stream(stream)


@pytest.mark.parametrize("nq,nk,dtype", [(300, 300, torch.float16), (2000, 100, torch.bfloat16)])
def test_graph_replays(cuda, nq, nk, dtype):
    """Forward and gradients captured together, without autograd, while an eager graph of the
    same tensors lives."""
    from hi3d_amd import attention

    q, k, v, dout = _tensors(nq, nk, 4, 2, 64, dtype)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    alive = attention.attend(*leaves)

    def both():
        with torch.no_grad():
            out, lse = attention.attend(*leaves, return_lse=True)
            return (out, *attention.attend_grad(*leaves, out, lse, dout))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        both()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for _ in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn_like(q))
        dout.copy_(torch.randn_like(dout))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, both()):
            assert torch.equal(a, b)
    assert alive.shape == q.shape
