"""What the torso's block does with its cache, without a GPU: plain stand-ins in the inputs' own
type (float64 here) for the two operators, so that the block's data flow is all that is tested.
Tolerance: sums of a few hundred float64 products, 1e-12 of values near one."""

from __future__ import annotations

import math

import pytest
import torch

TOL = dict(rtol=1e-12, atol=1e-12)


def _attend(q, k, v, cu_q=None, cu_k=None, *, lens_k=None, scale=None, causal=False, key_mask=None):
    """``attention.attend`` from its definition: one packed segment, or equal room."""
    assert cu_q is None and cu_k is None and k.shape == v.shape and k.shape[:-3] == q.shape[:-3]
    if q.dim() == 4:
        lens = [k.shape[1]] * k.shape[0] if lens_k is None else lens_k.tolist()
        assert key_mask is None or key_mask.shape == k.shape[:2]
        return torch.stack([_attend(q[b], k[b, :n], v[b, :n], causal=causal,
                                    key_mask=None if key_mask is None else key_mask[b, :n]) for b, n in enumerate(lens)])
    lq, lk, group = q.shape[0], k.shape[0], q.shape[1] // k.shape[1]
    assert key_mask is None or key_mask.shape == (lk,)
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    score = torch.einsum("ihd,jhd->hij", q, k) * (q.shape[-1] ** -0.5 if scale is None else scale)
    if causal:
        score = score.masked_fill(torch.arange(lk) > torch.arange(lq)[:, None] + (lk - lq), -math.inf)
    if key_mask is not None:
        score = score.masked_fill(~key_mask, -math.inf)
    return torch.einsum("hij,jhd->ihd", score.softmax(-1).nan_to_num(0.0), v)


def _turn(q, k, positions, freqs, *, layout):
    angle = (positions.double() @ freqs)[:, None]
    pad = q.shape[-1] // 2 - angle.shape[-1]
    wave = torch.nn.functional.pad(torch.polar(torch.ones_like(angle), angle), (0, pad), value=1.0)
    turned = lambda x: torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (-1, 2))) * wave).flatten(-2)  # noqa: E731
    assert layout == "interleaved"
    return turned(q), turned(k)


@pytest.fixture
def plain(monkeypatch):
    from hi3d_amd import attention, rotary

    monkeypatch.setattr(attention, "attend", _attend)
    monkeypatch.setattr(rotary, "rotate_qk", _turn)


def _block(causal=True, heads=4, key_heads=2):
    from hi3d_amd import torso

    torch.manual_seed(0)
    return torso.TokenAttention(8 * heads, heads, key_heads, axes=1, causal=causal, dtype=torch.float64)


def _cache(block, batch=1, length=40):
    from hi3d_amd import torso

    return torso.KeyValueCache(batch, length, block.key_heads, block.dim, torch.float64, device="cpu")


def _tokens(n, channels, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, channels, generator=g, dtype=torch.float64), torch.arange(n, dtype=torch.int32)[:, None]


@pytest.mark.parametrize("chunks", [(20,), (13, 7), (1, 1, 18), (5, 0, 15)])
def test_a_prompt_in_chunks(plain, chunks):
    """Every chunk sees what the cache holds already: the rows of one pass over all tokens."""
    block = _block()
    x, positions = _tokens(24, 32)
    want, cache, at, rows = block(x, positions), _cache(block), 0, []
    with torch.no_grad():
        for n in chunks:
            rows.append(block(x[at:at + n], positions[at:at + n], cache=cache))
            at += n
            assert cache.used == [at] == cache.lens.tolist()
        for i in range(at, 24):
            rows.append(block.step(x[i:i + 1], positions[i:i + 1], cache))
    torch.testing.assert_close(torch.cat(rows), want.detach(), **TOL)
    assert cache.used == [24]


def test_a_chunk_after_steps_and_without_a_causal_limit(plain):
    block = _block(causal=False)
    x, positions = _tokens(12, 32)
    cache = _cache(block)
    with torch.no_grad():
        block(x[:5], positions[:5], cache=cache)
        block.step(x[5:6], positions[5:6], cache)
        got = block(x[6:], positions[6:], cache=cache)
    torch.testing.assert_close(got, block(x, positions).detach()[6:], **TOL)


def test_gradients_of_a_chunk(plain):
    """The chunk's own keys take gradients; those that the cache held are constants, and keys
    that the cache takes later do not disturb the backward pass."""
    block = _block()
    x, positions = _tokens(20, 32)
    cache = _cache(block)
    with torch.no_grad():
        block(x[:9], positions[:9], cache=cache)
    leaf = x[9:].clone().requires_grad_(True)
    out = block(leaf, positions[9:], cache=cache)
    assert cache.used == [20] and not cache.k.requires_grad
    with torch.no_grad():
        block.step(x[:1], positions[:1], cache)
    got, = torch.autograd.grad(out.square().sum(), leaf)
    other = x[9:].clone().requires_grad_(True)
    whole = block(torch.cat([x[:9], other]), positions)[9:]
    want, = torch.autograd.grad(whole.square().sum(), other)
    torch.testing.assert_close(out, whole, **TOL)
    torch.testing.assert_close(got, want, **TOL)


@pytest.mark.parametrize("chunks", [(17,), (9, 8), (9, 0, 8)])
@pytest.mark.parametrize("late", [False, True])
def test_masked_prompts(plain, chunks, late):
    """Keys that a prompt's mask hides stay hidden from later parts and steps; ``late``: only the
    last part has a mask."""
    block = _block()
    x, positions = _tokens(22, 32)
    mask = torch.rand(17, generator=torch.Generator().manual_seed(2)) < 0.6
    if late:
        mask[:17 - chunks[-1]] = True
    shown = torch.cat([mask, torch.ones(5, dtype=torch.bool)])
    want, cache, at, rows = block(x, positions, key_mask=shown).detach(), _cache(block), 0, []
    with torch.no_grad():
        for i, n in enumerate(chunks):
            kw = {} if late and i + 1 < len(chunks) else dict(key_mask=mask[at:at + n])
            rows.append(block(x[at:at + n], positions[at:at + n], cache=cache, **kw))
            at += n
        for i in range(17, 20):
            rows.append(block.step(x[i:i + 1], positions[i:i + 1], cache))
        rows.append(block(x[20:], positions[20:], cache=cache))
    torch.testing.assert_close(torch.cat(rows), want, **TOL)


def test_gradients_over_masked_keys(plain):
    block = _block()
    x, positions = _tokens(20, 32)
    mask = torch.rand(20, generator=torch.Generator().manual_seed(3)) < 0.5
    cache = _cache(block)
    with torch.no_grad():
        block(x[:9], positions[:9], cache=cache, key_mask=mask[:9])
    leaf, other = (x[9:].clone().requires_grad_(True) for _ in range(2))
    got, = torch.autograd.grad(block(leaf, positions[9:], cache=cache, key_mask=mask[9:]).square().sum(), leaf)
    want, = torch.autograd.grad(block(torch.cat([x[:9], other]), positions, key_mask=mask)[9:].square().sum(), other)
    torch.testing.assert_close(got, want, **TOL)


def test_masks_of_several_sequences(plain):
    """A mask belongs to its sequence; the others see all their keys."""
    block = _block()
    x, positions = _tokens(11, 32)
    cache, mask = _cache(block, batch=2), torch.arange(10) % 3 != 1
    with torch.no_grad():
        _, k, v = block.project(x[:10], positions[:10])
        cache.extend(0, k[:6], v[:6])
        cache.extend(1, k, v, mask)
        got = block.step(x[[6, 10]], positions[[6, 10]], cache)
    torch.testing.assert_close(got[0], block(x[:7], positions[:7]).detach()[-1], **TOL)
    shown = torch.cat([mask, mask.new_ones(1)])
    torch.testing.assert_close(got[1], block(x, positions, key_mask=shown).detach()[-1], **TOL)


def _state(cache):
    return [x.clone() for x in (cache.k, cache.v, cache.lens)] + [list(cache.used), None if cache.mask is None else cache.mask.clone()]


def _same(a, b):
    return all(torch.equal(x, y) if torch.is_tensor(x) else x == y for x, y in zip(a, b))


@pytest.mark.parametrize("masked", [False, True])
def test_refused_keys_leave_the_cache_alone(masked):
    from hi3d_amd import torso

    cache = torso.KeyValueCache(3, 6, 2, 8, torch.float32, device="cpu")
    if masked:
        cache.extend(1, torch.ones(2, 2, 8), torch.ones(2, 2, 8), torch.tensor([True, False]))
    before, ones = _state(cache), torch.ones
    for k, v in [(ones(1, 2, 8), ones(1, 2, 8)), (ones(3, 1, 8), ones(3, 1, 8)), (ones(3, 2, 1), ones(3, 2, 1)),
                 (ones(3, 2, 8), ones(1, 2, 8)), (ones(2, 8), ones(2, 8)),
                 (ones(3, 2, 8, device="meta"), ones(3, 2, 8, device="meta")),
                 (ones(3, 2, 8), ones(3, 2, 16)), (ones(4, 2, 8), ones(4, 2, 8))]:
        with pytest.raises(ValueError, match="must be"):
            cache.append(k, v)
        assert _same(before, _state(cache))
    for k, v, mask in [(ones(4, 1, 8), ones(4, 1, 8), None), (ones(4, 2, 8), ones(1, 2, 8), None),
                       (ones(4, 2, 8), ones(4, 2, 1), None),
                       (ones(2, 8), ones(2, 8), None), (ones(1, 4, 2, 8), ones(1, 4, 2, 8), None),
                       (ones(4, 2, 8), ones(4, 2, 8), ones(4)), (ones(4, 2, 8), ones(4, 2, 8), ones(1, dtype=torch.bool)),
                       (ones(4, 2, 8), ones(4, 2, 8), ones(4, dtype=torch.bool, device="meta"))]:
        with pytest.raises(ValueError, match="must be"):
            cache.extend(2, k, v, mask)
        assert _same(before, _state(cache))
    for which in (-1, 3):
        with pytest.raises(ValueError, match="no sequence"):
            cache.extend(which, ones(1, 2, 8), ones(1, 2, 8))
        assert _same(before, _state(cache))


def test_refused_tokens_leave_the_cache_alone(plain):
    """Through the block: a token too few, a cache of another type or of other heads."""
    from hi3d_amd import torso

    block = _block()
    x, positions = _tokens(6, 32)
    for cache, batch in [(_cache(block, batch=3), 1), (_cache(block, batch=3), 2),
                         (torso.KeyValueCache(2, 9, 2, 8, torch.float32, device="cpu"), 2),
                         (torso.KeyValueCache(2, 9, 1, 8, torch.float64, device="cpu"), 2)]:
        before = _state(cache)
        with pytest.raises(ValueError, match="must be"):
            block.step(x[:batch], positions[:batch], cache)
        assert _same(before, _state(cache))
    for cache in (torso.KeyValueCache(1, 9, 2, 8, torch.float32, device="cpu"),
                  torso.KeyValueCache(1, 9, 1, 8, torch.float64, device="cpu")):
        before = _state(cache)
        with torch.no_grad(), pytest.raises(ValueError, match="must be"):
            block(x, positions, cache=cache)
        assert _same(before, _state(cache))


def test_a_cache_that_starts_again(plain):
    """A program that takes a cache again from its first key: the old mask hides nothing new."""
    block = _block()
    x, positions = _tokens(14, 32)
    cache = _cache(block)
    with torch.no_grad():
        block(x[:12], positions[:12], cache=cache, key_mask=torch.arange(12) % 2 == 0)
        cache.used[0] = 0
        cache.lens.zero_()
        rows = [block(x[:6], positions[:6], cache=cache)]
        rows += [block.step(x[i:i + 1], positions[i:i + 1], cache) for i in range(6, 9)]
        rows.append(block(x[9:], positions[9:], cache=cache))
    torch.testing.assert_close(torch.cat(rows), block(x, positions).detach(), **TOL)
