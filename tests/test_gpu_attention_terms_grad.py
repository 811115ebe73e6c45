"""Gradients of attention whose scores carry terms against float64 and against differences."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from terms_check import DTYPES, check, tensors, terms

pytestmark = pytest.mark.gpu

KINDS = ["cap", "slopes", "bias", "cap slopes bias"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [8, 32, 40, 64, 88, 96, 120, 128])
@pytest.mark.parametrize("kind", ["cap", "slopes", "bias"])
def test_head_sizes(cuda, kind, d, dtype):
    q, k, v, dout = tensors(150, 211, 4, 2, d, dtype)
    check(q, k, v, [150], [211], dout=dout, **terms(kind, 4, far=40))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 2), (2, 1), (31, 33), (32, 32), (63, 65), (65, 63), (127, 129), (257, 255),
                                   (300, 5), (5, 300), (1, 1000), (1000, 1), (517, 517)])
@pytest.mark.parametrize("kind", KINDS)
def test_lengths(cuda, kind, nq, nk, causal):
    q, k, v, dout = tensors(nq, nk, 2, 2, 64, torch.float16, gain=3.0)
    kw = terms(kind + (" prefix" if causal else ""), 2, far=30, causal=causal, longest=nk)
    check(q, k, v, [nq], [nk], dout=dout, causal=causal, **kw)


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
    q, k, v, dout = tensors(sum(lq), sum(lk or lq), 4, 2, 32, torch.bfloat16, seed=case)
    check(q, k, v, lq, lk, dout=dout, causal=causal,
          **terms(kind + (" prefix" if causal else ""), 4, len(lq), far=20, causal=causal))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hk", [(1, 1), (6, 2), (5, 1), (32, 8), (33, 33)])
def test_grouped_heads(cuda, hq, hk, kind):
    """Gradients of shared key heads, and of a bias that every query head has its own of."""
    q, k, v, dout = tensors(143, 143, hq, hk, 64, torch.float16)
    check(q, k, v, [143], dout=dout, causal=True, **terms(kind, hq, far=17, causal=True))


@pytest.mark.parametrize("far", [0, 1, 63, 64, 65, 200, 1024])
def test_reach_of_the_bias(cuda, far):
    q, k, v, dout = tensors(333, 400, 2, 1, 128, torch.bfloat16)
    bias = torch.randn((2 * far + 1, 2), generator=torch.Generator().manual_seed(far)).cuda()
    buckets = torch.arange(2 * far + 1, dtype=torch.int32).cuda()
    check(q, k, v, [333], [400], dout=dout, bias=bias, buckets=buckets.flip(0))
    check(q, k, v, [333], [400], dout=dout, bias=bias, buckets=buckets, causal=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_types_of_the_bias(cuda, dtype):
    q, k, v, dout = tensors(100, 100, 3, 3, 64, torch.float16)
    _, _, grads = check(q, k, v, [100], dout=dout, **terms("bias", 3, far=20, dtype=dtype))
    assert grads[3].dtype == dtype


@pytest.mark.parametrize("cap", [0.5, 30.0, 1024.0])
@pytest.mark.parametrize("gain", [0.01, 1.0, 60.0])
def test_caps(cuda, cap, gain):
    q, k, v, dout = tensors(70, 400, 2, 2, 64, torch.float16, gain=gain)
    check(q, k, v, [70], [400], dout=dout, cap=cap)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
@pytest.mark.parametrize("d", [64, 88])
def test_hidden_keys_may_hold_anything(cuda, d, fill, kind):
    lengths = [130, 64, 1, 200]
    n = sum(lengths)
    q, k, v, dout = tensors(n, n, 3, 3, d, torch.float16)
    mask = torch.rand(n, generator=torch.Generator().manual_seed(5)) < 0.6
    mask[130:194] = False
    mask[64:128] = False
    mask = mask.cuda()
    k[~mask], v[~mask] = fill, fill
    _, _, grads = check(q, k, v, lengths, mask=mask, dout=dout, **terms(kind, 3, far=20))
    assert not grads[1][~mask].any() and not grads[2][~mask].any()


def test_bias_that_hides(cuda):
    q, k, v, dout = tensors(150, 150, 2, 2, 64, torch.float16)
    bias = torch.tensor([[-float("inf"), -1e32], [0.5, -1e32], [-1e31, -1e32]]).cuda()
    buckets = torch.tensor([0] * 40 + [1] * 9 + [2] * 52, dtype=torch.int32).cuda()
    _, _, grads = check(q, k, v, [150], dout=dout, bias=bias, buckets=buckets, causal=True)
    assert not grads[3][0].any() and not grads[3][2].any() and not grads[3][:, 1].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
def test_gradient_of_lse(cuda, kind, dtype):
    q, k, v, dout = tensors(200, 300, 4, 2, 64, dtype)
    dlse = torch.randn((200, 4), generator=torch.Generator().manual_seed(9)).cuda()
    check(q, k, v, [200], [300], dout=dout, dlse=dlse, **terms(kind, 4, far=33))


@pytest.mark.parametrize("nq,nk,hq,hk,d", [(2500, 700, 4, 4, 64), (700, 2500, 4, 1, 128), (3000, 3000, 1, 1, 96)])
@pytest.mark.parametrize("kind", KINDS)
def test_long(cuda, kind, nq, nk, hq, hk, d):
    """Splits of the query rows for dk and dv, and more parts of the bias's gradient than one run."""
    q, k, v, dout = tensors(nq, nk, hq, hk, d, torch.bfloat16)
    check(q, k, v, [nq], [nk], dout=dout, **terms(kind, hq, far=128, count=32))


@pytest.mark.parametrize("hq,hk", [(32, 8), (24, 8)])
@pytest.mark.parametrize("causal,masked", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("kind", KINDS)
def test_wide_rows(cuda, kind, d, causal, masked, hq, hk):
    """Enough rows that they are neither split nor a few waves' work: the kernels that are built for one term,
    whose gradients take the output's digits past 16 bits; groups of heads that do and do not divide a tile."""
    q, k, v, dout = tensors(440, 440, hq, hk, d, torch.float16 if d % 64 else torch.bfloat16, gain=2.0)
    mask = (torch.rand(440, generator=torch.Generator().manual_seed(5)) < 0.7).cuda() if masked else None
    kw = terms(kind + (" prefix" if causal else ""), hq, 2, far=50, count=16, causal=causal, longest=200)
    check(q, k, v, [220, 220], dout=dout, causal=causal, mask=mask, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["cap", "slopes", "bias"])
def test_sharp_rows_keep_their_digits(cuda, kind, dtype):
    """Scores of standard deviation 4 over 400 keys leave a few keys to a row. Two roundings (of the score
    gradients, and of the result) of u each, independent: sqrt 2 of a single one's error, and 6 % for
    what is left of D's."""
    from oracle import attention_terms as oterms
    from terms_check import host, on_host

    q, k, v, dout = tensors(1200, 400, 16, 16, 64, dtype, gain=4.0)
    kw = terms(kind, 16, far=30, count=16)
    _, _, grads = check(q, k, v, [1200], [400], dout=dout, **kw)
    on = on_host(kw)
    off, single = [0.0] * 2, [0.0] * 2
    for h in range(16):
        f = oterms.head(host(q[:, h]), host(k[:, h]), host(v[:, h]), h, **on)
        r = oterms.head_grad(f, host(q[:, h]), host(dout[:, h]), 0.125, 0.0, 0.0, 0.0)
        for i, n in enumerate(("dq", "dk")):
            exact = torch.as_tensor(r[n])
            off[i] += float((grads[i][:, h].double().cpu() - exact).square().sum())
            single[i] += float((exact.to(dtype).double() - exact).square().sum())
    for a, b in zip(off, single):
        assert (a / b) ** 0.5 <= 1.5, (a / b) ** 0.5


def test_many_parts_of_the_bias(cuda):
    lengths = [48] * 700 + [11]
    q, k, v, dout = tensors(sum(lengths), sum(lengths), 2, 2, 32, torch.float16)
    check(q, k, v, lengths, dout=dout, **terms("bias", 2, far=60, count=16))


@pytest.mark.parametrize("kind", KINDS)
def test_against_differences(cuda, kind):
    """The derivative of sum(out * w) along random directions against central differences of a float64
    evaluation from the definition."""
    from oracle import attention_terms as oterms
    from terms_check import host, on_host

    q, k, v, dout = tensors(33, 50, 1, 1, 32, torch.float16)
    kw = terms(kind, 1, far=12)
    _, _, grads = check(q, k, v, [33], [50], dout=dout, **kw)
    on, w = on_host(kw), host(dout)[:, 0]
    rng = np.random.default_rng(0)
    values = [host(q)[:, 0], host(k)[:, 0], host(v)[:, 0]] + ([on["bias"]] if "bias" in kind else [])
    for which, value in enumerate(values):
        to = rng.standard_normal(value.shape)

        def at(step):
            x = [y + step * to if i == which else y for i, y in enumerate(values)]
            with_bias = dict(on, bias=x[3]) if len(x) > 3 else on
            return (oterms.head(x[0], x[1], x[2], 0, **with_bias)["out"] * w).sum()

        want = (at(1e-4) - at(-1e-4)) / 2e-4
        got = (host(grads[which]).reshape(value.shape) * to).sum()
        size = np.abs(host(grads[which]).reshape(value.shape) * to).sum()
        assert abs(got - want) <= 2.0 ** -8 * size + 1e-6, (which, got, want)


def test_only_some_gradients(cuda):
    from hi3d_amd import attention

    q, k, v, dout = tensors(120, 130, 4, 2, 64, torch.float16)
    kw = terms("cap slopes bias", 4, far=20)
    _, _, all_of = check(q, k, v, [120], [130], dout=dout, **kw)
    for wanted in ((0,), (1,), (2,), (3,), (0, 3), (1, 2)):
        leaves = [x.detach().requires_grad_(i in wanted) for i, x in enumerate((q, k, v, kw["bias"]))]
        out = attention.attend(*leaves[:3], **dict(kw, bias=leaves[3]))
        for i, g in zip(wanted, torch.autograd.grad(out, [leaves[i] for i in wanted], dout)):
            assert torch.equal(g, all_of[i])


def test_same_bits_every_time_and_in_replays(cuda):
    from hi3d_amd import attention

    q, k, v, dout = tensors(700, 700, 8, 2, 64, torch.bfloat16)
    kw = terms("cap slopes bias", 8, far=100, count=32)
    out, lse = attention.attend(q, k, v, return_lse=True, **kw)
    want = attention.attend_grad(q, k, v, out, lse, dout, **kw)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(attention.attend_grad(q, k, v, out, lse, dout, **kw), want))
    torch.cuda.current_stream().wait_stream(stream)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, m = attention.attend(q, k, v, return_lse=True, **kw)
        got = attention.attend_grad(q, k, v, o, m, dout, **kw)
    for _ in range(3):
        q.copy_(torch.randn_like(q)), dout.copy_(torch.randn_like(dout)), kw["bias"].mul_(0.7)
        graph.replay()
        torch.cuda.synchronize()
        out, lse = attention.attend(q, k, v, return_lse=True, **kw)
        want = attention.attend_grad(q, k, v, out, lse, dout, **kw)
        assert torch.equal(o, out) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_empty(cuda):
    from hi3d_amd import attention

    q, k, v, dout = tensors(10, 10, 2, 2, 64, torch.float16)
    kw = terms("bias", 2)
    for nq, nk in ((0, 10), (10, 0), (0, 0)):
        bias = kw["bias"].detach().requires_grad_(True)
        leaves = [x.detach().requires_grad_(True) for x in (q[:nq], k[:nk], v[:nk])]
        out = attention.attend(*leaves, bias=bias, buckets=kw["buckets"])
        grads = torch.autograd.grad(out, [*leaves, bias], dout[:nq])
        assert [g.shape for g in grads] == [x.shape for x in (*leaves, bias)] and not any(g.any() for g in grads)


def test_differentiable_once(cuda):
    from hi3d_amd import attention

    q, k, v, dout = tensors(10, 10, 2, 2, 64, torch.float16)
    bias = terms("bias", 2)["bias"].requires_grad_(True)
    out = attention.attend(q, k, v, bias=bias, buckets=terms("bias", 2)["buckets"])
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(out, bias, dout, create_graph=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steep", [30.0, 1e5])
def test_steep_slopes(cuda, steep, dtype):
    """Slopes that the score product's step cannot hold (in fp16, or for keys): one key a row."""
    q, k, v, dout = tensors(440, 440, 32, 8, 64, dtype)
    slopes = torch.full((32,), steep).cuda()
    slopes[::3] = 0.25
    check(q, k, v, [220, 220], dout=dout, slopes=slopes)
