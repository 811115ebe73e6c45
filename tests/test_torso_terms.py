"""What the torso's block does with terms and with caches that share their beginning, without a GPU: plain
stand-ins for the operators in float64, so that the block's data flow is all that is tested.
Tolerance: sums of a few hundred float64 products, 1e-12 of values near one."""

from __future__ import annotations

import pytest
import torch

from test_torso_cache import TOL, _attend, _cache, _tokens, _turn


def _with_terms(q, k, v, cu_q=None, cu_k=None, *, cap=None, slopes=None, bias=None, buckets=None, prefix=None, lens_k=None,
                key_mask=None, **kw):
    """``attention.attend`` where only the order of keys matters: terms are taken into the queries' scale."""
    terms = dict(cap=cap, slopes=slopes, bias=bias, buckets=buckets, prefix=prefix)
    if q.dim() == 4:
        lens = [k.shape[1]] * len(q) if lens_k is None else lens_k.tolist()
        return torch.stack([_with_terms(q[b], k[b, :n], v[b, :n], key_mask=None if key_mask is None else key_mask[b, :n],
                                        **terms, **kw) for b, n in enumerate(lens)])
    scale = q.shape[-1] ** -0.5 * (1 if cap is None else cap) * (1 if bias is None else float(bias.sum()) + 2.0)
    return _attend(q, k, v, cu_q, cu_k, scale=scale, key_mask=key_mask, **kw)


def _shared(q, pk, pv, k, v, *, lens_k=None, causal=False, shared_mask=None, key_mask=None, **terms):
    """``attention.attend_shared`` by concatenation, sequence by sequence."""
    rows = []
    for b in range(q.shape[0]):
        n = k.shape[1] if lens_k is None else int(lens_k[b])
        ones = [torch.ones(m, dtype=torch.bool) for m in (pk.shape[0], n)]
        mask = torch.cat([ones[0] if shared_mask is None else shared_mask, ones[1] if key_mask is None else key_mask[b, :n]])
        rows.append(_with_terms(q[b], torch.cat([pk, k[b, :n]]), torch.cat([pv, v[b, :n]]), causal=causal, key_mask=mask, **terms))
    return torch.stack(rows)


@pytest.fixture
def plain(monkeypatch):
    from hi3d_amd import attention, rotary

    monkeypatch.setattr(attention, "attend", _with_terms)
    monkeypatch.setattr(attention, "attend_shared", _shared)
    monkeypatch.setattr(rotary, "rotate_qk", _turn)


def _block(causal=True, **kw):
    from hi3d_amd import torso

    torch.manual_seed(0)
    return torso.TokenAttention(32, 4, 2, axes=1, causal=causal, dtype=torch.float64, **kw)


def _caches(block, batch=1):
    from hi3d_amd import torso

    shared = _cache(block)
    return shared, torso.KeyValueCache(batch, 40, 2, 8, torch.float64, device="cpu", shared=shared)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("masked", [False, True])
def test_a_prompt_behind_a_shared_one(plain, causal, masked):
    """In parts and steps: the rows of a cache that holds all of it."""
    block = _block(causal, cap=0.5)
    x, positions = _tokens(24, 32)
    mask = (torch.rand(24, generator=torch.Generator().manual_seed(3)) < 0.7) if masked else None
    part = lambda a, b: None if mask is None else mask[a:b]  # noqa: E731
    alone = _cache(block)
    shared, cache = _caches(block)
    with torch.no_grad():
        block(x[:10], positions[:10], cache=alone, key_mask=part(0, 10))
        block(x[:10], positions[:10], cache=shared, key_mask=part(0, 10))
        for a, b in ((10, 14), (14, 20)):
            got, want = (block(x[a:b], positions[a:b], cache=c, key_mask=part(a, b)) for c in (cache, alone))
            torch.testing.assert_close(got, want, **TOL)
        for i in range(20, 24):
            got, want = (block.step(x[i:i + 1], positions[i:i + 1], c) for c in (cache, alone))
            torch.testing.assert_close(got, want, **TOL)
    assert shared.used == [10] and cache.used == [14]


@pytest.mark.parametrize("masked", [False, True])
def test_gradients_behind_a_shared_prompt(plain, masked):
    block = _block(cap=0.5, buckets=4, far=5)
    x, positions = _tokens(20, 32)
    mask = (torch.rand(20, generator=torch.Generator().manual_seed(3)) < 0.7) if masked else None
    shared, cache = _caches(block)
    alone = _cache(block)
    grads = []
    for first, rest in ((alone, alone), (shared, cache)):
        with torch.no_grad():
            block(x[:9], positions[:9], cache=first, key_mask=None if mask is None else mask[:9])
        leaf = x[9:].clone().requires_grad_(True)
        out = block(leaf, positions[9:], cache=rest, key_mask=None if mask is None else mask[9:])
        grads.append(torch.autograd.grad(out.square().sum(), leaf)[0])
    torch.testing.assert_close(*grads, **TOL)


def test_steps_of_several_sequences(plain):
    block = _block()
    x, positions = _tokens(12, 32)
    shared, cache = _caches(block, 3)
    with torch.no_grad():
        block(x[:6], positions[:6], cache=shared)
        for i in range(2):
            got = block.step(x[6 + 3 * i:9 + 3 * i], positions[6:9], cache)
    assert cache.used == [2, 2, 2] and got.shape == (3, 32)
    for b in range(3):
        alone = _cache(block)
        with torch.no_grad():
            block(x[:6], positions[:6], cache=alone)
            for i in range(2):
                want = block.step(x[6 + 3 * i + b:7 + 3 * i + b], positions[6 + b:7 + b], alone)
        torch.testing.assert_close(got[b:b + 1], want, **TOL)


def test_terms_of_the_block():
    from hi3d_amd import attention

    block = _block(cap=30.0, slopes=True, buckets=8, far=20)
    terms = block.terms(torch.device("cpu"))
    assert terms["cap"] == 30.0 and torch.equal(terms["slopes"], attention.head_slopes(4, "cpu"))
    assert torch.equal(terms["buckets"], attention.relative_buckets(8, 20, causal=True, device="cpu"))
    assert terms["bias"] is block.relative_bias and block.relative_bias.shape == (8, 4)
    assert "relative_bias" in dict(block.named_parameters())
    block.half()
    assert block.terms(torch.device("cpu"))["slopes"].dtype == torch.float32
    assert _block().terms(torch.device("cpu")) == {} and _block().relative_bias is None


def test_refusals(plain):
    from hi3d_amd import torso

    for kw in (dict(cap=0.0), dict(cap=5000.0), dict(buckets=3, causal=False), dict(buckets=8, far=2)):
        with pytest.raises(ValueError):
            _block(**kw)
    block = _block()
    x, positions = _tokens(4, 32)
    prefix = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="prefix"):
        block(x, positions, cache=_cache(block), prefix=prefix)
    with pytest.raises(ValueError, match="prefix"):
        _block(causal=False)(x, positions, prefix=prefix)
    shared, cache = _caches(block)
    for wrong in (cache, torso.KeyValueCache(2, 4, 2, 8, torch.float64, device="cpu"),
                  torso.KeyValueCache(1, 4, 2, 8, torch.float32, device="cpu"),
                  torso.KeyValueCache(1, 4, 1, 8, torch.float64, device="cpu")):
        with pytest.raises(ValueError, match="share"):
            torso.KeyValueCache(1, 4, 2, 8, torch.float64, device="cpu", shared=wrong)


def test_terms_first_used_in_inference_mode_serve_gradients_later():
    block = _block(slopes=True, buckets=8, far=20)
    with torch.inference_mode():
        terms, freqs = block.terms(torch.device("meta")), block.frequencies(torch.device("meta"))
    assert not any(t.is_inference() for t in (freqs, terms["slopes"], terms["buckets"]))
    assert block.terms(torch.device("meta"))["slopes"] is terms["slopes"]
