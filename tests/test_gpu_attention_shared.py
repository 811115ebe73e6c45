"""Attention over keys that a batch shares, in front of each sequence's own, against float64 and against
attention over the concatenated keys."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import attention_terms as oterms
from terms_check import DTYPES, check_rows, host, on_host, tensors, terms

pytestmark = pytest.mark.gpu


def _problem(batch, new, own, shared, hq, hk, d, dtype, gain=1.0):
    q, k, v, _ = tensors(batch * new, batch * own, hq, hk, d, dtype, gain=gain)
    _, pk, pv, _ = tensors(0, shared, hq, hk, d, dtype, seed=8)
    return q.reshape(batch, new, hq, d), pk, pv, k.reshape(batch, own, hk, d), v.reshape(batch, own, hk, d)


def _check(q, pk, pv, k, v, lens=None, causal=False, shared_mask=None, key_mask=None, scale=None, **kw):
    from hi3d_amd import attention

    batch, new, hq, d = q.shape
    own, hk, shared = k.shape[1], k.shape[2], pk.shape[0]
    lens_k = None if lens is None else torch.tensor(lens, dtype=torch.int32).cuda()
    out, lse = attention.attend_shared(q, pk, pv, k, v, lens_k=lens_k, causal=causal, shared_mask=shared_mask, key_mask=key_mask,
                                       scale=scale, return_lse=True, **kw)
    on, sm, km = on_host(kw), host(shared_mask), host(key_mask)
    for b in range(batch):
        n = own if lens is None else min(max(lens[b], 0), own)
        r = np.arange(-shared, n)[None, :] - (np.arange(new)[:, None] + n - new)
        seen = np.ones((new, shared + n), bool)
        if causal:
            seen &= (r <= 0) | (np.arange(-shared, n) < 0)
        if sm is not None:
            seen[:, :shared] &= sm > 0
        if km is not None:
            seen[:, shared:] &= km[b, :n] > 0
        for h in range(hq):
            g = h // (hq // hk)
            kk, vv = (np.concatenate([host(x[:, g]), host(y[b, :n, g])]) for x, y in ((pk, k), (pv, v)))
            f = oterms.head(host(q[b, :, h]), kk, vv, h, scale, r=r, seen=seen, **on)
            check_rows(out[b, :, h], lse[b, :, h], f, q.dtype, f"out of sequence {b} head {h}")
    return out, lse


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [8, 32, 40, 64, 88, 96, 120, 128])
@pytest.mark.parametrize("kind", ["", "cap slopes bias"])
def test_head_sizes(cuda, kind, d, dtype):
    _check(*_problem(3, 1, 70, 300, 4, 2, d, dtype), lens=[70, 1, 33], **terms(kind, 4, far=40))


@pytest.mark.parametrize("batch,new,own,shared,hq,hk", [
    (1, 1, 1, 1, 1, 1), (1, 1, 50, 3000, 8, 8), (40, 1, 20, 5000, 4, 1), (3, 4, 64, 63, 6, 2), (70, 1, 5, 65, 1, 1),
    (2, 33, 40, 257, 4, 2), (5, 3, 700, 20, 33, 33), (2, 200, 300, 1000, 2, 2), (33, 2, 17, 129, 8, 1)])
@pytest.mark.parametrize("kind", ["", "cap", "slopes", "bias"])
@pytest.mark.parametrize("causal", [False, True])
def test_sizes(cuda, causal, kind, batch, new, own, shared, hq, hk):
    lens = [(own * (i + 1)) // batch for i in range(batch)]
    _check(*_problem(batch, new, own, shared, hq, hk, 64, torch.float16, gain=2.0), lens=lens, causal=causal,
           **terms(kind, hq, far=30, count=16))


def test_without_shared_or_own_keys(cuda):
    from hi3d_amd import attention

    q, pk, pv, k, v = _problem(3, 2, 40, 50, 4, 2, 64, torch.bfloat16)
    _check(q, pk[:0], pv[:0], k, v, lens=[40, 0, 7])
    _check(q, pk, pv, k[:, :0], v[:, :0])
    _check(q, pk, pv, k, v, lens=[0, 0, 0], causal=True)
    out, lse = attention.attend_shared(q, pk[:0], pv[:0], k[:, :0], v[:, :0], return_lse=True)
    assert not out.any() and bool(torch.isneginf(lse).all())
    assert attention.attend_shared(q[:0], pk, pv, k[:0], v[:0]).shape == (0, 2, 4, 64)
    assert attention.attend_shared(q[:, :0], pk, pv, k, v).shape == (3, 0, 4, 64)


@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
def test_masks(cuda, fill):
    q, pk, pv, k, v = _problem(3, 2, 130, 200, 4, 2, 88, torch.float16)
    g = torch.Generator().manual_seed(1)
    shared_mask, key_mask = (torch.rand(200, generator=g) < 0.5).cuda(), (torch.rand((3, 130), generator=g) < 0.5).cuda()
    shared_mask[64:128], key_mask[1] = False, False
    pk[~shared_mask], pv[~shared_mask], k[~key_mask], v[~key_mask] = fill, fill, fill, fill
    k[0, 100:], v[0, 100:] = fill, fill
    _check(q, pk, pv, k, v, lens=[100, 130, 5], causal=True, shared_mask=shared_mask, key_mask=key_mask)
    none = torch.zeros(200, dtype=torch.bool).cuda()
    out, _ = _check(q, pk, pv, k, v, lens=[100, 130, 5], shared_mask=none, key_mask=key_mask)
    assert not out[1].any()


def test_nearly_the_bits_of_concatenated_keys(cuda):
    """The same probabilities, rounded around other references: within two roundings of each other."""
    from hi3d_amd import attention

    q, pk, pv, k, v = _problem(6, 1, 90, 700, 8, 2, 128, torch.bfloat16)
    lens = torch.tensor([90, 3, 1, 50, 64, 65], dtype=torch.int32).cuda()
    got = attention.attend_shared(q, pk, pv, k, v, lens_k=lens)
    kk, vv = (torch.cat([x.expand(6, -1, -1, -1), y], 1) for x, y in ((pk, k), (pv, v)))
    want = attention.attend(q, kk, vv, lens_k=lens + 700)
    size = attention.attend(q, kk, vv.abs(), lens_k=lens + 700).float()
    assert bool(((got.float() - want.float()).abs() <= 4 * 2.0 ** -8 * size).all())


def test_views(cuda):
    from hi3d_amd import attention

    q, pk, pv, k, v = _problem(3, 2, 40, 50, 4, 2, 64, torch.float16)
    want = attention.attend_shared(q, pk, pv, k, v, causal=True)
    cache = torch.randn((50, 5, 64), device="cuda").half()
    cache[:, :2], cache[:, 2:4] = pk, pv
    both = torch.randn((3, 60, 4, 64), device="cuda").half()
    both[:, 7:47, :2], both[:, 7:47, 2:] = k, v
    wide = torch.randn((3, 5, 9, 64), device="cuda").half()
    wide[:, 1:3, 2:6] = q
    got = attention.attend_shared(wide[:, 1:3, 2:6], cache[:, :2], cache[:, 2:4], both[:, 7:47, :2], both[:, 7:47, 2:], causal=True)
    assert torch.equal(got, want)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(attention.attend_shared(turned, pk, pv, k, v, causal=True), want)


def test_replays(cuda):
    from hi3d_amd import attention

    q, pk, pv, k, v = _problem(6, 1, 90, 4000, 8, 2, 128, torch.bfloat16)
    lens = torch.tensor([90, 3, 1, 50, 64, 65], dtype=torch.int32).cuda()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        attention.attend_shared(q, pk, pv, k, v, lens_k=lens)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attention.attend_shared(q, pk, pv, k, v, lens_k=lens)
    for _ in range(3):
        q.copy_(torch.randn_like(q)), lens.copy_(torch.randint_like(lens, 1, 91))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, attention.attend_shared(q, pk, pv, k, v, lens_k=lens))
