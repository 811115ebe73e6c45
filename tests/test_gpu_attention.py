"""Attention and its gradients against float64.

Tolerances follow the roundings. With u half a step of the type and e = 2^-24:

* a score (fp32, d products) is off by at most (d + 4) e times ``reach`` = scale sum |q k|,
  and an exponential adds 4 e: a probability is off by a relative ``pe`` = 2 (d + 4) e reach +
  (16 + keys) e (numerator and sum);
* the probabilities are rounded to the type for their product: u each, and in fp16 an
  absolute 2^-25 where they are below its normal range;
* the output is rounded once.

The gradients' bounds (``oracle.attention.backward``) carry the same through their sums."""

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


def _expect(q, k, v, cu_q, cu_k, scale, causal, mask):
    return oattention.forward(_np(q), _np(k), _np(v), oattention.spans(cu_q), oattention.spans(cu_k), scale, causal,
                              None if mask is None else mask.cpu().numpy())


def _p_error(want, d, keys):
    return 2 * (d + 4) * E * want["reach"] + (16 + keys) * E


def _out_room(want, dtype, d, keys):
    pe = _p_error(want, d, keys)[..., None]
    return (U[dtype] + pe) * want["size"] + TINY[dtype] * want["vsum"] + U[dtype] * np.abs(want["out"]) + 2 * TINY[dtype]


def _within(got, want, room, what):
    got = _np(got)
    assert got.shape == want.shape
    assert np.isfinite(got).all(), f"{what} is not finite"
    off = np.abs(got - want) - room
    assert (off <= 0).all(), f"{what}: {np.max(np.abs(got - want) / np.maximum(room, 1e-300))} of the room"


def _check_forward(out, lse, q, k, v, cu_q, cu_k, scale=None, causal=False, mask=None):
    d, keys = q.shape[-1], max([b - a for a, b in oattention.spans(cu_k)] + [0])
    want = _expect(q, k, v, cu_q, cu_k, scale, causal, mask)
    _within(out, want["out"], _out_room(want, q.dtype, d, keys), "out")
    if lse is not None:
        got, empty = _np(lse), np.isneginf(want["lse"])
        assert np.array_equal(np.isneginf(got), empty)
        off = np.abs(np.where(empty, 0, got) - np.where(empty, 0, want["lse"]))
        room = _p_error(want, d, keys) + 4 * E * np.abs(np.where(empty, 0, want["lse"])) + 8 * E
        assert (off <= room).all(), np.max(off / room)
    return want


def _tensors(nq, nk, hq, hk, d, dtype, seed=0, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    make = lambda n, h, s: (s * torch.randn((n, h, d), generator=g)).to(dtype).cuda()  # noqa: E731
    return make(nq, hq, gain), make(nk, hk, gain), make(nk, hk, 1.0)


def _cu(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [8, 32, 40, 64, 88, 96, 120, 128])
def test_head_sizes(cuda, d, dtype):
    from hi3d_amd import attention

    q, k, v = _tensors(150, 211, 4, 2, d, dtype)
    out, lse = attention.attend(q, k, v, return_lse=True)
    _check_forward(out, lse, q, k, v, [0, 150], [0, 211])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 2), (2, 1), (31, 33), (32, 32), (63, 65), (64, 64), (65, 63), (127, 129),
                                   (128, 128), (257, 255), (300, 5), (5, 300), (1, 1000), (517, 517)])
def test_lengths(cuda, nq, nk, causal, dtype):
    """Causal queries past the keys (nq > nk) see nothing and give zeros."""
    from hi3d_amd import attention

    q, k, v = _tensors(nq, nk, 2, 2, 64, dtype)
    out, lse = attention.attend(q, k, v, causal=causal, return_lse=True)
    _check_forward(out, lse, q, k, v, [0, nq], [0, nk], causal=causal)
    if causal and nq > nk:
        assert not out[:nq - nk].any()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 4), (6, 2), (5, 1), (32, 8), (33, 33)])
def test_grouped_heads(cuda, hq, hk, causal):
    from hi3d_amd import attention

    q, k, v = _tensors(143, 143, hq, hk, 64, torch.bfloat16)
    _check_forward(attention.attend(q, k, v, causal=causal), None, q, k, v, [0, 143], [0, 143], causal=causal)


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
def test_segments(cuda, case, causal):
    from hi3d_amd import attention

    lq, lk = RAGGED[case]
    cu_q, cu_k = _cu(lq), _cu(lk if lk is not None else lq)
    q, k, v = _tensors(int(cu_q[-1]), int(cu_k[-1]), 4, 2, 32, torch.float16, seed=case)
    kw = {} if lk is None else {"cu_k": attention.offsets(lk)}
    out, lse = attention.attend(q, k, v, attention.offsets(lq), causal=causal, return_lse=True, **kw)
    _check_forward(out, lse, q, k, v, cu_q, cu_k, causal=causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -float("inf"), 65504.0])
@pytest.mark.parametrize("d", [64, 88])
def test_hidden_keys_may_hold_anything(cuda, d, fill, dtype):
    from hi3d_amd import attention

    lengths = [130, 64, 1, 200]
    cu = _cu(lengths)
    n = int(cu[-1])
    q, k, v = _tensors(n, n, 3, 3, d, dtype)
    mask = torch.rand(n, generator=torch.Generator().manual_seed(5)) < 0.6
    mask[130:194] = False  # a segment without keys
    mask[64:128] = False  # a whole tile of a segment
    mask = mask.cuda()
    clean = attention.attend(q, k, v, attention.offsets(lengths), key_mask=mask, return_lse=True)
    _check_forward(*clean, q, k, v, cu, cu, mask=mask)
    assert not clean[0][130:194].any()
    k[~mask], v[~mask] = fill, fill
    for a, b in zip(clean, attention.attend(q, k, v, attention.offsets(lengths), key_mask=mask, return_lse=True)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("causal", [False, True])
def test_mask_with_groups_and_long_rows(cuda, causal):
    from hi3d_amd import attention

    q, k, v = _tensors(190, 900, 8, 2, 128, torch.bfloat16)
    mask = (torch.rand(900, generator=torch.Generator().manual_seed(6)) < 0.3).cuda()
    out, lse = attention.attend(q, k, v, causal=causal, key_mask=mask, return_lse=True)
    _check_forward(out, lse, q, k, v, [0, 190], [0, 900], causal=causal, mask=mask)


def test_large_scores(cuda):
    """Scores of a few hundred: a running maximum that jumps late in the row."""
    from hi3d_amd import attention

    q, k, v = _tensors(70, 400, 2, 2, 64, torch.float16, gain=4.0)
    k[390:] *= 3
    _check_forward(attention.attend(q, k, v), None, q, k, v, [0, 70], [0, 400])
    _check_forward(attention.attend(q, k, v, scale=0.7), None, q, k, v, [0, 70], [0, 400], scale=0.7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,cache,hq,hk,d,lens", [
    (1, 1030, 33, 33, 64, None), (3, 777, 32, 8, 128, [777, 1, 400]), (2, 5000, 4, 1, 96, [4999, 0]),
    (5, 64, 8, 8, 32, [0, 64, 63, 1, 200]), (1, 20011, 16, 2, 88, None)])
def test_single_tokens_over_a_cache(cuda, batch, cache, hq, hk, d, lens, dtype):
    from hi3d_amd import attention

    q, k, v = _tensors(batch, batch * cache, hq, hk, d, dtype)
    use = [min(n, cache) for n in lens] if lens else [cache] * batch
    cu_q = _cu([1] * batch)
    parts = [slice(b * cache, b * cache + n) for b, n in enumerate(use)]
    kk, vv = (torch.cat([x[p] for p in parts]) for x in (k, v))
    lens_k = None if lens is None else torch.tensor(lens, dtype=torch.int32).cuda()
    shape = (batch, cache, hk, d)
    for b, n in enumerate(use):  # what lies past the keys in use is never read into a result
        k[b * cache + n:(b + 1) * cache] = float("nan")
        v[b * cache + n:(b + 1) * cache] = float("nan")
    out, lse = attention.attend(q[:, None], k.reshape(shape), v.reshape(shape), lens_k=lens_k, return_lse=True)
    assert out.shape == (batch, 1, hq, d)
    _check_forward(out[:, 0], lse[:, 0], q, kk, vv, cu_q, _cu(use))


def test_views(cuda):
    from hi3d_amd import attention

    g = torch.Generator().manual_seed(2)
    qkv = torch.randn((333, 7 + 7 + 7, 64), generator=g).half().cuda()
    q, k, v = qkv[:, :7], qkv[:, 7:14], qkv[:, 14:]
    want = attention.attend(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(attention.attend(q, k, v), want)
    heads_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(attention.attend(*heads_first), want)
    values_apart = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    assert torch.equal(attention.attend(*values_apart), want)
    odd = torch.empty(333 * (21 * 64 + 3) + 1, dtype=torch.float16, device="cuda")[1:].as_strided((333, 21, 64), (1347, 64, 1))
    odd.copy_(qkv)
    assert torch.equal(attention.attend(odd[:, :7], odd[:, 7:14], odd[:, 14:]), want)
    one = torch.randn((333, 1, 64), generator=g).half().cuda()
    spread = one.expand(333, 7, 64)
    assert torch.equal(attention.attend(q, spread, spread), attention.attend(q, one, one))
    dense = qkv.reshape(3, 111, 21, 64).transpose(0, 1).contiguous().transpose(0, 1)
    got = attention.attend(dense[:, :, :7], dense[:, :, 7:14], dense[:, :, 14:])
    assert torch.equal(got.reshape(333, 7, 64), attention.attend(q, k, v, attention.offsets([111] * 3)))


def test_empty(cuda):
    from hi3d_amd import attention

    q, k, v = _tensors(10, 10, 2, 2, 64, torch.float16)
    assert attention.attend(q[:0], k, v).shape == (0, 2, 64)
    out, lse = attention.attend(q, k[:0], v[:0], return_lse=True)
    assert not out.any() and bool(torch.isneginf(lse).all())
    assert attention.attend(q[:0], k[:0], v[:0], attention.offsets([])).shape == (0, 2, 64)
    assert attention.attend(q[:0], k[:0], v[:0], attention.offsets([0, 0])).shape == (0, 2, 64)


def test_same_bits_every_time_and_on_another_stream(cuda):
    from hi3d_amd import attention

    q, k, v = _tensors(1, 9000, 16, 2, 128, torch.bfloat16)
    want = attention.attend(q, k, v)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            assert torch.equal(attention.attend(q, k, v), want)
    torch.cuda.current_stream().wait_stream(stream)


@pytest.mark.parametrize("nq,nk", [(300, 300), (1, 4000)])
def test_graph_replays(cuda, nq, nk):
    from hi3d_amd import attention

    q, k, v = _tensors(nq, nk, 8, 2, 64, torch.float16)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        attention.attend(q, k, v, return_lse=True)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = attention.attend(q, k, v, return_lse=True)
    for _ in range(3):
        q.copy_(torch.randn_like(q))
        graph.replay()
        torch.cuda.synchronize()
        a, b = attention.attend(q, k, v, return_lse=True)
        assert torch.equal(out, a) and torch.equal(lse, b)


def test_long_cache_past_32_bit_offsets(cuda):
    """4.4e9 values of keys: byte and element offsets pass 32 bits."""
    from hi3d_amd import attention

    n, hk, d = 1 << 22, 8, 128
    kv = torch.empty((1, n + 77, hk, d), dtype=torch.bfloat16, device="cuda")
    kv.normal_()
    q = torch.randn((1, 1, hk, d), device="cuda").to(torch.bfloat16)
    lens = torch.tensor([n + 77], dtype=torch.int32, device="cuda")
    out = attention.attend(q, kv, kv, lens_k=lens)[0, 0]
    for h in (0, 7):
        x = kv[0, :, h].double()
        s = x @ q[0, 0, h].double() * d ** -0.5
        p = torch.softmax(s, 0)
        want, size = (p @ x), (p @ x.abs())
        # sums of 4 million terms in fp32 add their own rounding: 2^-24 times a few thousand
        # (64 terms a lane and tile, then tiles, lanes and splits)
        room = U[torch.bfloat16] * (size + want.abs()) + 2.0 ** -12 * size
        assert bool(((out[h].double() - want).abs() <= room).all())
