"""The torso's block with terms in its scores, its prompts and steps over caches that share their
beginning, against the block in float64. Tolerances as in ``test_gpu_torso``: root mean square
errors below 8 half steps of the type for outputs, 16 for gradients (32 for those of the bias, sums
of score gradients of both signs that are rounded nowhere but in q, k, v and dout)."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_torso import U, _rms

pytestmark = pytest.mark.gpu

KINDS = {"cap": dict(cap=2.0), "slopes": dict(slopes=True), "bias": dict(buckets=16, far=40),
         "all": dict(cap=3.0, slopes=True, buckets=8, far=20)}


def _block(kind, dtype, heads=4, key_heads=2, dim=64, causal=True):
    from hi3d_amd import torso

    torch.manual_seed(1)
    block = torso.TokenAttention(dim * heads, heads, key_heads, axes=1, causal=causal, dtype=dtype, device="cuda", **KINDS[kind])
    if block.relative_bias is not None:
        torch.nn.init.normal_(block.relative_bias)
    return block


def _tokens(n, channels, dtype, seed=4):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, channels, generator=g).to(dtype).cuda(), torch.arange(n, dtype=torch.int32).cuda()[:, None]


def _plain(block, x, positions, lengths, prefix=None):
    """The block in float64 from its definition."""
    w = {n: p.detach().double().requires_grad_(True) for n, p in block.named_parameters()}
    h, hk, d, terms = block.heads, block.key_heads, block.dim, block.terms(x.device)
    y = x @ w["qkv.weight"].T + w["qkv.bias"]
    q, k, v = y.view(len(x), h + 2 * hk, d).split([h, hk, hk], 1)
    t = (positions.double() @ block.frequencies(x.device))[:, None]
    turn = lambda z: torch.stack([z[..., 0::2] * t.cos() - z[..., 1::2] * t.sin(),  # noqa: E731
                                  z[..., 0::2] * t.sin() + z[..., 1::2] * t.cos()], -1).flatten(-2)
    q, k, v = turn(q), turn(k).repeat_interleave(h // hk, 1), v.repeat_interleave(h // hk, 1)
    outs, at = [], 0
    for i, n in enumerate(lengths):
        s = slice(at, at + n)
        at += n
        score = torch.bmm(q[s].transpose(0, 1), k[s].permute(1, 2, 0).contiguous()) * d ** -0.5
        place = torch.arange(n, device=x.device)
        r = place - place[:, None]
        if "cap" in terms:
            score = terms["cap"] * torch.tanh(score / terms["cap"])
        if "slopes" in terms:
            score = score - terms["slopes"].double()[:, None, None] * r.abs()
        if "bias" in terms:
            far = len(terms["buckets"]) // 2
            score = score + w["relative_bias"].T[:, terms["buckets"].long()[r.clamp(-far, far) + far]]
        if block.causal:
            score = score.masked_fill((r > 0) & (place >= (0 if prefix is None else prefix[i])), -math.inf)
        outs.append(torch.bmm(score.softmax(-1), v[s].transpose(0, 1).contiguous()).transpose(0, 1).reshape(n, -1))
    return torch.cat(outs) @ w["out.weight"].T + w["out.bias"], w


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_training_step(cuda, kind, causal, dtype):
    from hi3d_amd import attention

    block, lengths = _block(kind, dtype, causal=causal), [130, 1, 303]
    x, positions = _tokens(434, 256, dtype)
    prefix = [40, 0, 100] if causal else None
    dout = _tokens(434, 256, dtype, seed=5)[0]
    x.requires_grad_(True)
    out = block(x, positions, attention.offsets(lengths),
                prefix=None if prefix is None else torch.tensor(prefix, dtype=torch.int32).cuda())
    out.backward(dout)
    xd = x.detach().double().requires_grad_(True)
    want, w = _plain(block, xd, positions, lengths, prefix)
    want.backward(dout.double())
    assert _rms(out.double() - want) <= 8 * U[dtype] * _rms(want)
    assert _rms(x.grad.double() - xd.grad) <= 16 * U[dtype] * _rms(xd.grad)
    for name, p in block.named_parameters():
        room = 32 if name == "relative_bias" else 16
        assert _rms(p.grad.double() - w[name].grad) <= room * U[dtype] * _rms(w[name].grad), name


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", KINDS)
def test_prompt_and_steps(cuda, kind, dtype):
    from hi3d_amd import torso

    block = _block(kind, dtype)
    x, positions = _tokens(210, 256, dtype)
    want = _plain(block, x.double(), positions, [210])[0].detach()
    cache, rows = torso.KeyValueCache(1, 220, 2, 64, dtype), []
    with torch.no_grad():
        for a, b in ((0, 130), (130, 131), (131, 200)):
            rows.append(block(x[a:b], positions[a:b], cache=cache))
        for i in range(200, 210):
            rows.append(block.step(x[i:i + 1], positions[i:i + 1], cache))
    rows = torch.cat(rows).double()
    assert _rms(rows - want) <= 8 * U[dtype] * _rms(want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", KINDS)
def test_sequences_that_share_their_beginning(cuda, kind, dtype):
    """Three sequences after one prompt: steps of all three, a prompt part of one of them, and its gradient."""
    from hi3d_amd import torso

    block = _block(kind, dtype)
    x, positions = _tokens(150, 256, dtype)
    more, _ = _tokens(3 * 9, 256, dtype, seed=6)
    more = more.view(3, 9, 256)
    places = torch.arange(150, 159, dtype=torch.int32).cuda()[:, None]
    shared = torso.KeyValueCache(1, 150, 2, 64, dtype)
    cache, rows = torso.KeyValueCache(3, 20, 2, 64, dtype, shared=shared), []
    with torch.no_grad():
        block(x, positions, cache=shared)
        for i in range(9):
            rows.append(block.step(more[:, i], places[i].expand(3, 1), cache))
    rows = torch.stack(rows, 1).double()
    for b in range(3):
        want = _plain(block, torch.cat([x, more[b]]).double(), torch.cat([positions, places]), [159])[0].detach()[150:]
        assert _rms(rows[b] - want) <= 8 * U[dtype] * _rms(want)
    one = torso.KeyValueCache(1, 20, 2, 64, dtype, shared=shared)
    with torch.no_grad():
        parts = [block(more[1, a:b], places[a:b], cache=one) for a, b in ((0, 4), (4, 9))]
    want = _plain(block, torch.cat([x, more[1]]).double(), torch.cat([positions, places]), [159])[0].detach()[150:]
    assert _rms(torch.cat(parts).double() - want) <= 8 * U[dtype] * _rms(want)
    one = torso.KeyValueCache(1, 20, 2, 64, dtype, shared=shared)
    leaf = more[1].clone().requires_grad_(True)
    out = block(leaf, places, cache=one)
    assert _rms(out.detach().double() - want) <= 8 * U[dtype] * _rms(want)
    grad, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    xd = more[1].double().requires_grad_(True)
    whole = _plain(block, torch.cat([x.double(), xd]), torch.cat([positions, places]), [159])[0][150:]
    exact, = torch.autograd.grad(whole, xd, torch.ones_like(whole))
    assert _rms(grad.double() - exact) <= 16 * U[dtype] * _rms(exact)


def test_masked_prompts_that_are_shared(cuda):
    from hi3d_amd import torso

    block = _block("cap", torch.float16)
    x, positions = _tokens(60, 256, torch.float16)
    mask = torch.rand(60, generator=torch.Generator().manual_seed(2)).cuda() < 0.6
    mask[-10:] = True
    alone = torso.KeyValueCache(1, 80, 2, 64)
    shared = torso.KeyValueCache(1, 50, 2, 64)
    cache = torso.KeyValueCache(1, 30, 2, 64, shared=shared)
    with torch.no_grad():
        block(x[:50], positions[:50], cache=alone, key_mask=mask[:50])
        want = [block(x[50:], positions[50:], cache=alone, key_mask=mask[50:]), block.step(x[:1], positions[:1], alone)]
        block(x[:50], positions[:50], cache=shared, key_mask=mask[:50])
        got = [block(x[50:], positions[50:], cache=cache, key_mask=mask[50:]), block.step(x[:1], positions[:1], cache)]
    for a, b in zip(got, want):
        assert _rms(a.double() - b.double()) <= 8 * U[torch.float16] * _rms(b)


def test_captured_steps_over_a_shared_beginning(cuda):
    """The step's two operators in a graph: replays see the cache's keys and lengths as they are then."""
    from hi3d_amd import attention, torso

    block = _block("all", torch.bfloat16)
    x, positions = _tokens(150, 256, torch.bfloat16)
    shared = torso.KeyValueCache(1, 150, 2, 64, torch.bfloat16)
    cache = torso.KeyValueCache(3, 20, 2, 64, torch.bfloat16, shared=shared)
    with torch.no_grad():
        block(x, positions, cache=shared)
        block.step(x[:3], positions[:3], cache)
        q = torch.randn(3, 1, 4, 64, device="cuda").bfloat16()
        call = lambda: attention.attend_shared(q, *shared_k, cache.k, cache.v, lens_k=cache.lens, **block.terms(q.device))  # noqa: E731
        shared_k = cache.shared_keys()[:2]
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            call()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for i in range(3):
            block.step(x[3 * i:3 * i + 3], positions[3 * i:3 * i + 3], cache)
            q.copy_(torch.randn_like(q))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, call())


def test_gradients_after_a_first_call_in_inference_mode():
    grads = []
    for first in (True, False):
        block = _block("all", torch.bfloat16)
        x, positions = _tokens(70, block.heads * block.dim, torch.bfloat16)
        if first:
            with torch.inference_mode():
                block(x, positions)
        block(x, positions).float().square().sum().backward()
        grads.append([p.grad for p in block.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*grads))
