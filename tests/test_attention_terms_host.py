"""Attention with terms in its scores, without a GPU: what is refused before anything is launched, the
bucket maps, the workspace queries of the C entries, and the oracle against direct sums."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from oracle import attention_terms as oterms


def _qkv(n=4, heads=4, key_heads=2, dim=64, dtype=torch.float16):
    return [torch.randn(n, h, dim).to(dtype) for h in (heads, key_heads, key_heads)]


def _bias(count=4, heads=4, dtype=torch.float32):
    return torch.zeros(count, heads, dtype=dtype), torch.tensor([0, 1, 2], dtype=torch.int32)


@pytest.mark.parametrize("kw,match", [
    (dict(cap=0.0), "cap"), (dict(cap=-1.0), "cap"), (dict(cap=1025.0), "cap"), (dict(cap=math.inf), "cap"),
    (dict(cap=math.nan), "cap"),
    (dict(slopes=torch.ones(2)), "slopes"), (dict(slopes=torch.ones(4).half()), "slopes"), (dict(slopes=torch.ones(4, 1)), "slopes"),
    (dict(bias=_bias()[0]), "buckets"), (dict(buckets=_bias()[1]), "bias"),
    (dict(bias=torch.zeros(4, 2), buckets=_bias()[1]), "bias"), (dict(bias=torch.zeros(4), buckets=_bias()[1]), "bias"),
    (dict(bias=torch.zeros(0, 4), buckets=_bias()[1]), "bias"), (dict(bias=torch.zeros(4, 4).double(), buckets=_bias()[1]), "bias"),
    (dict(bias=_bias()[0], buckets=torch.zeros(4, dtype=torch.int32)), "buckets"),
    (dict(bias=_bias()[0], buckets=torch.zeros(3, dtype=torch.int64)), "buckets"),
    (dict(bias=_bias()[0], buckets=torch.zeros(2051, dtype=torch.int32)), "buckets"),
    (dict(bias=_bias()[0], buckets=torch.zeros(3, 1, dtype=torch.int32)), "buckets"),
    (dict(prefix=torch.zeros(1, dtype=torch.int32)), "causal"),
    (dict(prefix=torch.zeros(2, dtype=torch.int32), causal=True), "prefix"),
    (dict(prefix=torch.zeros(1), causal=True), "prefix"),
])
def test_refusals(kw, match):
    from hi3d_amd import attention

    q, k, v = _qkv()
    with pytest.raises(ValueError, match=match):
        attention.attend(q, k, v, **kw)
    with pytest.raises(ValueError, match=match):
        attention.attend_grad(q, k, v, q, torch.zeros(4, 4), q, **kw)


def test_host_tensors_are_refused():
    from hi3d_amd import attention

    q, k, v = _qkv()
    for kw in (dict(cap=3.0), dict(slopes=torch.ones(4)), dict(zip(("bias", "buckets"), _bias())),
               dict(prefix=torch.zeros(1, dtype=torch.int32), causal=True)):
        with pytest.raises(ValueError, match="ROCm GPU only"):
            attention.attend(q, k, v, **kw)


def test_slopes_that_wait_for_a_gradient_are_refused():
    from hi3d_amd import attention

    q, k, v = _qkv()
    slopes = torch.ones(4, requires_grad=True)
    with pytest.raises(NotImplementedError, match="constants"):
        attention.attend(q, k, v, slopes=slopes)
    with torch.no_grad(), pytest.raises(ValueError, match="ROCm GPU only"):
        attention.attend(q, k, v, slopes=slopes)


def test_tangents_are_refused():
    from hi3d_amd import attention

    q, k, v = _qkv()
    bias, buckets = _bias()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(bias, torch.ones_like(bias))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            attention.attend(q, k, v, bias=dual, buckets=buckets)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            attention.attend_grad(q, k, v, q, torch.zeros(4, 4), q, bias=dual, buckets=buckets)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            attention.attend_shared(q[None], k, v, k[None], v[None], bias=dual, buckets=buckets)


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(4, 4, 64).half()), "batch"),
    (dict(shared_k=torch.zeros(5, 1, 64).half()), "shared_k"), (dict(shared_v=torch.zeros(5, 2, 32).half()), "shared_v"),
    (dict(shared_k=torch.zeros(5, 2, 64).bfloat16()), "shared_k"), (dict(shared_v=torch.zeros(6, 2, 64).half()), "differ"),
    (dict(shared_mask=torch.ones(6, dtype=torch.bool)), "shared_mask"), (dict(shared_mask=torch.ones(5)), "shared_mask"),
    (dict(cap=2000.0), "cap"), (dict(lens_k=torch.zeros(2, dtype=torch.int32)), "lens_k"),
    (dict(shared_k=torch.zeros(1, 2, 64).half().expand(1 << 31, 2, 64)), "2\\^31"),
])
def test_shared_refusals(kw, match, monkeypatch):
    from hi3d_amd import _lib, attention

    monkeypatch.setattr(_lib, "require_gpu", lambda *t: torch.device("cpu"))  # the checks behind it are this test's
    given = dict(q=torch.zeros(3, 2, 4, 64).half(), shared_k=torch.zeros(5, 2, 64).half(), shared_v=torch.zeros(5, 2, 64).half(),
                 k=torch.zeros(3, 7, 2, 64).half(), v=torch.zeros(3, 7, 2, 64).half())
    with pytest.raises(ValueError, match=match):
        attention.attend_shared(**{**given, **kw})


def test_shared_keys_form_no_gradients():
    from hi3d_amd import attention

    q, k = torch.zeros(3, 2, 4, 64).half(), torch.zeros(3, 7, 2, 64).half()
    shared = torch.zeros(5, 2, 64).half()
    with pytest.raises(NotImplementedError, match="gradients"):
        attention.attend_shared(q.requires_grad_(True), shared, shared, k, k)
    with torch.no_grad(), pytest.raises(ValueError, match="ROCm GPU only"):
        attention.attend_shared(q, shared, shared, k, k)


@pytest.mark.parametrize("count,far,causal", [(32, 128, False), (32, 128, True), (4, 1024, False), (2, 5, True), (64, 400, False),
                                              (64, 700, True), (16, 48, False)])
def test_buckets(count, far, causal):
    """Each side: a bucket a distance, then by the logarithm of the distance; borders in whole numbers."""
    from hi3d_amd import attention

    got = attention.relative_buckets(count, far, causal=causal, device="cpu")
    side = count if causal else count // 2
    near = side // 2
    assert got.dtype == torch.int32 and got.shape == (2 * far + 1,)
    for r in range(-far, far + 1):
        d, later = abs(r), r > 0
        if later and causal:
            assert got[r + far] == 0
            continue
        place = int(got[r + far]) - (side if later else 0)
        if d < near:
            assert place == d
        else:
            rest, n = side - near, place - near
            assert 0 <= n < rest
            assert d ** rest * near ** n >= far ** n * near ** rest
            assert n == rest - 1 or d ** rest * near ** (n + 1) < far ** (n + 1) * near ** rest
    assert len(set(got.tolist())) <= count and int(got.max()) < count


@pytest.mark.parametrize("count,far,causal", [(3, 10, False), (2, 10, False), (1, 10, True), (0, 10, True), (32, 8, False),
                                              (32, 1025, False), (32, 0, False)])
def test_buckets_refusals(count, far, causal):
    from hi3d_amd import attention

    with pytest.raises(ValueError):
        attention.relative_buckets(count, far, causal=causal, device="cpu")


def test_slopes():
    from hi3d_amd import attention

    assert torch.equal(attention.head_slopes(8, "cpu"), torch.tensor([2.0 ** -i for i in range(1, 9)]))
    assert attention.head_slopes(33, "cpu").shape == (33,)
    with pytest.raises(ValueError):
        attention.head_slopes(0, "cpu")


def _desc(attention, nq=100, nk=100, hq=4, hk=2, dim=64, causal=0, scale=0.125, dtype=1):
    d = attention._Desc()
    d.q, d.k, d.v = 4096, 8192, 12288  # never read by a size query
    d.strides[:] = [nq * hq * dim, hq * dim, dim, nk * hk * dim, hk * dim, dim, nk * hk * dim, hk * dim, dim]
    d.total_q, d.total_k, d.batch, d.len_q, d.len_k = nq, nk, 1, nq, nk
    d.heads_q, d.heads_k, d.dim, d.dtype, d.causal, d.scale = hq, hk, dim, dtype, causal, scale
    return d


@pytest.mark.parametrize("kw,terms,match", [
    ({}, dict(cap=-1.0), "cap"), ({}, dict(cap=2000.0), "cap"), ({}, dict(cap=float("nan")), "cap"),
    (dict(scale=1e-38), dict(slopes=4096), "scale"), ({}, dict(prefix=4096), "causal"),
    ({}, dict(bias=4096, bucket_map=4096, buckets=4, far=3, bias_dtype=5), "bias"),
    ({}, dict(bias=4096, buckets=4, far=3), "null"), ({}, dict(bias=4096, bucket_map=4096, buckets=0, far=3), "buckets"),
    ({}, dict(bias=4096, bucket_map=4096, buckets=4, far=-1), "1024"), ({}, dict(bias=4096, bucket_map=4096, buckets=4, far=1025), "1024"),
    (dict(hq=64, hk=1), dict(bias=4096, bucket_map=4096, buckets=4, far=200), "query heads"),
])
def test_c_entries_refuse(kw, terms, match):
    from hi3d_amd import _lib, attention

    d, t, out = _desc(attention, **kw), attention._TermsDesc(**terms), ctypes.c_int64(7)
    for name, more in (("hi3d_attention_terms_workspace", (None,)), ("hi3d_attention_terms_backward_workspace", ())):
        with pytest.raises(ValueError, match=match):
            _lib.call(name, ctypes.byref(d), ctypes.byref(t), *more, ctypes.byref(out))


def test_c_entries_refuse_null_and_small_workspaces():
    from hi3d_amd import _lib, attention

    d, t, out = _desc(attention), attention._TermsDesc(), ctypes.c_int64(7)
    with pytest.raises(ValueError, match="terms"):
        _lib.call("hi3d_attention_terms_workspace", ctypes.byref(d), None, None, ctypes.byref(out))
    with pytest.raises(ValueError, match="null"):
        _lib.call("hi3d_attention_terms_workspace", ctypes.byref(d), ctypes.byref(t), None, None)
    with pytest.raises(ValueError, match="workspace"):
        _lib.call("hi3d_attention_terms_backward", ctypes.byref(d), ctypes.byref(t), 4096, None, 4096, 4096, None, 4096, 4096, 4096,
                  None, 4096, 1, None)
    with pytest.raises(ValueError, match="no bias"):
        _lib.call("hi3d_attention_terms_backward", ctypes.byref(d), ctypes.byref(t), 4096, None, 4096, 4096, None, 4096, 4096, 4096,
                  4096, 4096, 1 << 40, None)


@pytest.mark.parametrize("change,match", [
    (dict(strides=(7, 64, 128, 64)), "multiples of 8"), (dict(strides=(1 << 23, 64, 128, 64)), "2\\^23"),
    (dict(len=-1), "sizes"), (dict(k=None), "null"), (dict(v=4104), "aligned")])
def test_shared_c_entries_refuse(change, match):
    from hi3d_amd import _lib, attention

    d, t, out = _desc(attention), attention._TermsDesc(), ctypes.c_int64(7)
    s = attention._SharedDesc(4096, 4096, None, (128, 64, 128, 64), 50)
    for name, value in change.items():
        if name == "strides":
            s.strides[:] = value
        else:
            setattr(s, name, value)
    with pytest.raises(ValueError, match=match):
        _lib.call("hi3d_attention_shared_workspace", ctypes.byref(d), ctypes.byref(t), ctypes.byref(s), ctypes.byref(out))
    d.cu_q = 4096
    with pytest.raises(ValueError, match="offsets"):
        _lib.call("hi3d_attention_shared_workspace", ctypes.byref(d), ctypes.byref(t), ctypes.byref(s), ctypes.byref(out))


def test_which_rows_keep_their_rest():
    """Only rows of attend_kernel that are not split: few rows, short segments and parts do not."""
    from hi3d_amd import _lib, attention

    t, bytes_, kept = attention._TermsDesc(cap=5.0), ctypes.c_int64(0), ctypes.c_int32(7)
    for kw, want in ((dict(nq=20000, nk=20000), 1), (dict(nq=300, nk=300), 0), (dict(nq=40, nk=40), 0), (dict(nq=1, nk=90000), 0),
                     (dict(nq=0, nk=10), 0)):
        d = _desc(attention, **kw)
        _lib.call("hi3d_attention_terms_workspace", ctypes.byref(d), ctypes.byref(t), ctypes.byref(kept), ctypes.byref(bytes_))
        assert kept.value == want, kw


def test_oracle_against_direct_sums():
    rng = np.random.default_rng(0)
    lq, lk, d, heads = 5, 9, 8, 2
    q, k, v, do = rng.standard_normal((lq, d)), rng.standard_normal((lk, d)), rng.standard_normal((lk, d)), rng.standard_normal((lq, d))
    slopes, bias, buckets = np.array([0.5, 0.25]), rng.standard_normal((3, heads)), np.array([2, 1, 0, 1, 2])

    def scores(q, k, bias, h=1, prefix=2):
        s = np.full((lq, lk), -np.inf)
        for i in range(lq):
            for j in range(lk):
                r = j - (i + lk - lq)
                if r <= 0 or j < prefix:
                    s[i, j] = 2.0 * math.tanh(q[i] @ k[j] / math.sqrt(d) / 2.0) - slopes[h] * abs(r) + bias[buckets[max(-2, min(2, r)) + 2], h]
        return s

    def out(q, k, v, bias):
        s = scores(q, k, bias)
        p = np.exp(s - s.max(1, keepdims=True))
        return p / p.sum(1, keepdims=True) @ v

    f = oterms.head(q, k, v, 1, causal=True, prefix=2, cap=2.0, slopes=slopes, bias=bias, buckets=buckets)
    assert np.allclose(f["out"], out(q, k, v, bias), atol=1e-12)
    s = scores(q, k, bias)
    assert np.allclose(f["lse"], np.log(np.exp(s).sum(1)), atol=1e-12)
    g = oterms.head_grad(f, q, do, d ** -0.5, 0.0, 0.0, 0.0)
    dbias = np.zeros((3, heads))
    np.add.at(dbias[:, 1], buckets[np.clip(oterms.positions(lq, lk), -2, 2) + 2], g["ds"])
    at = [q, k, v, bias]
    for which, got in enumerate((g["dq"], g["dk"], g["dv"], dbias)):
        to = rng.standard_normal(at[which].shape)
        step = lambda e: (out(*[x + e * to if i == which else x for i, x in enumerate(at)]) * do).sum()  # noqa: B023, E731
        assert abs((step(1e-5) - step(-1e-5)) / 2e-5 - (got * to).sum()) < 1e-7
