"""Attention whose scores carry terms, forward and single tokens, against float64."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import attention_terms as oterms
from terms_check import DTYPES, check, check_rows, ends, host, on_host, tensors, terms

pytestmark = pytest.mark.gpu

KINDS = ["cap", "slopes", "bias", "cap slopes bias"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [8, 32, 40, 64, 88, 96, 120, 128])
@pytest.mark.parametrize("kind", ["cap", "slopes", "bias"])
def test_head_sizes(cuda, kind, d, dtype):
    q, k, v, _ = tensors(150, 211, 4, 2, d, dtype)
    check(q, k, v, [150], [211], **terms(kind, 4, far=40))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 2), (2, 1), (31, 33), (32, 32), (63, 65), (64, 64), (65, 63), (127, 129),
                                   (257, 255), (300, 5), (5, 300), (1, 1000), (517, 517)])
@pytest.mark.parametrize("kind", KINDS)
def test_lengths(cuda, kind, nq, nk, causal):
    q, k, v, _ = tensors(nq, nk, 2, 2, 64, torch.float16, gain=3.0)
    kw = terms(kind + (" prefix" if causal else ""), 2, far=30, causal=causal, longest=nk)
    check(q, k, v, [nq], [nk], causal=causal, **kw)


RAGGED = [
    ([48] * 9 + [29], None),
    ([1, 0, 2, 700, 0, 0, 33, 64, 128, 1], None),
    ([0, 0, 5], [0, 7, 0]),
    ([300, 20, 0, 77], [3, 0, 90, 400]),
    ([17] * 200, None),
    ([(7 * i) % 90 for i in range(150)], [(11 * i) % 70 for i in range(150)]),
    ([17] * 100 + [900] + [5] * 100, None),
    ([9] * 60 + [300], [5] * 60 + [1200]),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", range(len(RAGGED)))
def test_segments(cuda, case, kind, causal):
    lq, lk = RAGGED[case]
    q, k, v, _ = tensors(sum(lq), sum(lk or lq), 4, 2, 32, torch.bfloat16, seed=case)
    check(q, k, v, lq, lk, causal=causal, **terms(kind + (" prefix" if causal else ""), 4, len(lq), far=20, causal=causal))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hk", [(1, 1), (6, 2), (5, 1), (32, 8), (33, 33)])
def test_grouped_heads(cuda, hq, hk, kind):
    q, k, v, _ = tensors(143, 143, hq, hk, 64, torch.bfloat16)
    check(q, k, v, [143], causal=True, **terms(kind, hq, far=17, causal=True))


@pytest.mark.parametrize("nq,nk,hq,hk,d", [(600, 700, 8, 8, 32), (9000, 300, 8, 8, 64), (700, 3000, 2, 2, 128), (40, 3000, 2, 1, 96),
                                           (1100, 1100, 1, 1, 64), (33, 9000, 1, 1, 64), (50, 20000, 1, 1, 128)])
@pytest.mark.parametrize("kind", KINDS)
def test_tiles(cuda, kind, nq, nk, hq, hk, d):
    """Every tile rule: 256 and 128 rows, 64 and 32 of one wave, eight waves, and splits of the keys."""
    q, k, v, _ = tensors(nq, nk, hq, hk, d, torch.float16, gain=2.0)
    check(q, k, v, [nq], [nk], **terms(kind, hq, far=128, count=32))


@pytest.mark.parametrize("far", [0, 1, 31, 63, 64, 65, 200, 1024])
def test_reach_of_the_bias(cuda, far):
    """Buckets of their own for every position, so that a place off by one shows."""
    q, k, v, _ = tensors(333, 400, 2, 1, 64, torch.float16)
    g = torch.Generator().manual_seed(far)
    bias = torch.randn((2 * far + 1, 2), generator=g).cuda()
    buckets = torch.arange(2 * far + 1, dtype=torch.int32).cuda()
    check(q, k, v, [333], [400], bias=bias, buckets=buckets)
    check(q, k, v, [333], [400], bias=bias, buckets=buckets.flip(0), causal=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_types_of_the_bias(cuda, dtype):
    q, k, v, _ = tensors(100, 100, 3, 3, 64, torch.float16)
    check(q, k, v, [100], **terms("bias", 3, far=20, dtype=dtype))


@pytest.mark.parametrize("cap", [1e-3, 0.5, 30.0, 1024.0])
@pytest.mark.parametrize("gain", [0.01, 1.0, 60.0])
def test_caps(cuda, cap, gain):
    """Far below the bend, at it and past it, where the derivative is zero and scores are +-cap."""
    q, k, v, _ = tensors(70, 400, 2, 2, 64, torch.float16, gain=gain)
    check(q, k, v, [70], [400], cap=cap)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -float("inf"), 65504.0])
@pytest.mark.parametrize("d", [64, 88])
def test_hidden_keys_may_hold_anything(cuda, d, fill, kind):
    from hi3d_amd import attention

    lengths = [130, 64, 1, 200]
    n = sum(lengths)
    q, k, v, _ = tensors(n, n, 3, 3, d, torch.float16)
    mask = torch.rand(n, generator=torch.Generator().manual_seed(5)) < 0.6
    mask[130:194] = False  # a segment without keys
    mask[64:128] = False  # a whole tile of a segment
    mask = mask.cuda()
    kw = terms(kind, 3, far=20)
    clean = check(q, k, v, lengths, mask=mask, **kw)
    assert not clean[0][130:194].any()
    k[~mask], v[~mask] = fill, fill
    got = attention.attend(q, k, v, attention.offsets(lengths), key_mask=mask, return_lse=True, **kw)
    for a, b in zip(clean, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("low", [-float("inf"), torch.finfo(torch.float32).min, -1e31])
def test_bias_that_hides(cuda, low):
    """Buckets that no query sees, so that rows near the ends see no key at all."""
    q, k, v, _ = tensors(150, 150, 2, 2, 64, torch.bfloat16)
    bias = torch.zeros((5, 2))
    bias[:, 0] = torch.tensor([low, 0.5, low, 0.25, low])
    bias[:, 1] = low
    buckets = torch.tensor([0] * 40 + [1] * 9 + [2] * 3 + [3] * 9 + [4] * 40, dtype=torch.int32).cuda()
    out, lse, _ = check(q, k, v, [150], bias=bias.cuda(), buckets=buckets, causal=True)
    assert not out[:, 1].any() and bool(torch.isneginf(lse[:, 1]).all()) and not out[0, 0].any()


def test_lowest_number_of_a_short_type_is_a_number(cuda):
    """-65504 in fp16 is a bias like others: keys that all carry it share the row."""
    q, k, v, _ = tensors(40, 40, 1, 1, 64, torch.float16)
    bias = torch.full((1, 1), -65504.0, dtype=torch.float16).cuda()
    check(q, k, v, [40], bias=bias, buckets=torch.zeros(3, dtype=torch.int32).cuda())


def test_buckets_outside_the_table_count_as_the_nearest(cuda):
    q, k, v, _ = tensors(40, 40, 2, 2, 64, torch.float16)
    bias = torch.randn((3, 2), generator=torch.Generator().manual_seed(1)).cuda()
    buckets = torch.tensor([-5, 0, 1, 2, 99], dtype=torch.int32).cuda()
    check(q, k, v, [40], bias=bias, buckets=buckets)


@pytest.mark.parametrize("prefix", [-3, 0, 1, 64, 65, 129, 200, 100000, 1 << 32, -(1 << 33) + 7])
def test_prefix(cuda, prefix):
    q, k, v, _ = tensors(260, 200, 4, 2, 64, torch.float16)
    check(q, k, v, [130, 130], [70, 130], causal=True, prefix=torch.tensor([prefix, prefix], dtype=torch.int64).cuda())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,cache,hq,hk,d,lens", [
    (1, 1030, 33, 33, 64, None), (3, 777, 32, 8, 128, [777, 1, 400]), (2, 5000, 4, 1, 96, [4999, 0]),
    (5, 64, 8, 8, 32, [0, 64, 63, 1, 200]), (1, 20011, 16, 2, 88, None)])
@pytest.mark.parametrize("kind", KINDS)
def test_single_tokens_over_a_cache(cuda, kind, batch, cache, hq, hk, d, lens, dtype):
    from hi3d_amd import attention

    q, k, v, _ = tensors(batch, batch * cache, hq, hk, d, dtype, gain=2.0)
    use = [min(n, cache) for n in lens] if lens else [cache] * batch
    lens_k = None if lens is None else torch.tensor(lens, dtype=torch.int32).cuda()
    kw = terms(kind, hq, far=128, count=32, causal=True)
    k, v = (x.reshape(batch, cache, hk, d) for x in (k, v))
    for b, n in enumerate(use):  # what lies past the keys in use is never read into a result
        k[b, n:], v[b, n:] = float("nan"), float("nan")
    out, lse = attention.attend(q[:, None], k, v, lens_k=lens_k, return_lse=True, **kw)
    on = on_host(kw)
    for b, n in enumerate(use):
        for h in range(hq):
            g = h // (hq // hk)
            f = oterms.head(host(q[b, h])[None], host(k[b, :n, g]), host(v[b, :n, g]), h, **on)
            check_rows(out[b, :, h], lse[b, :, h], f, dtype)


def test_far_distances_keep_their_digits(cuda):
    """Slopes of 2^-8 over 70,000 keys: the constant part of a tile is formed apart from the score."""
    q, k, v, _ = tensors(2, 70001, 8, 1, 64, torch.bfloat16)
    check(q, k, v, [2], [70001], **terms("slopes", 8))


def test_same_bits_on_another_stream_and_in_replays(cuda):
    from hi3d_amd import attention

    q, k, v, _ = tensors(300, 4000, 8, 2, 64, torch.float16)
    kw = terms("cap slopes bias", 8, far=100, count=32)
    want = attention.attend(q, k, v, **kw)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            assert torch.equal(attention.attend(q, k, v, **kw), want)
    torch.cuda.current_stream().wait_stream(stream)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attention.attend(q, k, v, **kw)
    for i in range(3):
        q.copy_(torch.randn_like(q))
        kw["bias"].mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, attention.attend(q, k, v, **kw))


def test_terms_that_add_nothing(cuda):
    """A prefix of zero, slopes and a bias of zeros: plain attention, by the kernels with terms. (Not its bits:
    a row's reference is a multiply-add with zero here and one with the room below it there, an ulp apart.)"""
    q, k, v, _ = tensors(500, 500, 4, 2, 64, torch.float16)
    zero = torch.zeros(1, dtype=torch.int32).cuda()
    check(q, k, v, [500], causal=True, prefix=zero)
    check(q, k, v, [500], slopes=torch.zeros(4).cuda(), bias=torch.zeros((1, 4)).cuda(), buckets=zero)


def test_rows_outside_the_offsets_give_zeros(cuda):
    from hi3d_amd import attention

    q, k, v, _ = tensors(100, 100, 2, 2, 64, torch.float16)
    cu = torch.tensor([10, 50, 70], dtype=torch.int32).cuda()
    kw = terms("cap slopes bias", 2, far=8)
    out = attention.attend(q, k, v, cu, causal=True, prefix=torch.tensor([3, 4], dtype=torch.int32).cuda(), **kw)
    assert not out[:10].any() and not out[70:].any()
    inner = attention.attend(q[10:70], k[10:70], v[10:70], cu - 10, causal=True,
                             prefix=torch.tensor([3, 4], dtype=torch.int32).cuda(), **kw)
    assert torch.equal(out[10:70], inner)


def test_empty(cuda):
    from hi3d_amd import attention

    q, k, v, _ = tensors(10, 10, 2, 2, 64, torch.float16)
    kw = terms("cap slopes bias", 2)
    assert attention.attend(q[:0], k, v, **kw).shape == (0, 2, 64)
    out, lse = attention.attend(q, k[:0], v[:0], return_lse=True, **kw)
    assert not out.any() and bool(torch.isneginf(lse).all())
    assert attention.attend(q[:0], k[:0], v[:0], attention.offsets([]), **kw).shape == (0, 2, 64)
    assert np.array_equal(ends([]), [0])


@pytest.mark.parametrize("nq,nk,hq,hk,d", [(16400, 130, 32, 32, 64), (5600, 200, 96, 32, 32)])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_rows_of_two_blocks_a_wave(cuda, kind, masked, nq, nk, hq, hk, d):
    """256 rows to a workgroup, with heads that do and do not agree between a lane's two rows; some heads are
    checked."""
    from hi3d_amd import attention

    q, k, v, _ = tensors(nq, nk, hq, hk, d, torch.float16, gain=2.0)
    mask = (torch.rand(nk, generator=torch.Generator().manual_seed(7)) < 0.6).cuda() if masked else None
    kw = terms(kind, hq, far=50, count=16)
    out, lse = attention.attend(q, k, v, key_mask=mask, return_lse=True, **kw)
    on, m = on_host(kw), None if mask is None else mask.cpu().numpy()
    for h in (0, 1, 2, hq - 1):
        g = h // (hq // hk)
        f = oterms.head(host(q[:, h]), host(k[:, g]), host(v[:, g]), h, mask=m, **on)
        check_rows(out[:, h], lse[:, h], f, torch.float16)
