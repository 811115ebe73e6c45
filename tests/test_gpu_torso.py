"""The torso's attention block: operators together, against the same in float64.

Tolerance: every stage rounds once to the type (projection, rotation, probabilities, attention,
output projection; their gradients again on the way back), each by half a step u at most: root
mean square errors below 8 u of the outputs' and 16 u of the gradients' root mean square."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _plain(block, x, positions, lengths, causal):
    """The block in float64 from its definition."""
    w = {n: p.detach().double().requires_grad_(True) for n, p in block.named_parameters()}
    h, hk, d = block.heads, block.key_heads, block.dim
    y = x @ w["qkv.weight"].T + w["qkv.bias"]
    q, k, v = y.view(len(x), h + 2 * hk, d).split([h, hk, hk], 1)
    freqs = block.frequencies(x.device)
    t = (positions.double() @ freqs)[:, None]
    cos, sin = t.cos(), t.sin()

    def turn(z):
        rot = 2 * freqs.shape[1]
        a, b = z[..., 0:rot:2], z[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        return torch.cat([turned, z[..., rot:]], -1)

    q, k = turn(q), turn(k).repeat_interleave(h // hk, 1)
    v = v.repeat_interleave(h // hk, 1)
    outs, at = [], 0
    for n in lengths:
        s = slice(at, at + n)
        at += n
        score = torch.bmm(q[s].transpose(0, 1), k[s].permute(1, 2, 0).contiguous()) * d ** -0.5
        if causal:
            score = score.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), -math.inf)
        outs.append(torch.bmm(score.softmax(-1), v[s].transpose(0, 1).contiguous()).transpose(0, 1).reshape(n, -1))
    return torch.cat(outs) @ w["out.weight"].T + w["out.bias"], w


def _rms(x):
    return x.double().square().mean().sqrt()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,key_heads,causal", [(3, 3, False), (4, 2, True)])
def test_training_step(cuda, heads, key_heads, causal, dtype):
    from hi3d_amd import attention, torso

    torch.manual_seed(0)
    block = torso.TokenAttention(64 * heads, heads, key_heads, causal=causal, dtype=dtype, device="cuda")
    lengths = [130, 1, 203]
    x = torch.randn(sum(lengths), 64 * heads, device="cuda").to(dtype).requires_grad_(True)
    positions = torch.randint(0, 512, (sum(lengths), 3), device="cuda", dtype=torch.int32)
    dout = torch.randn(sum(lengths), 64 * heads, device="cuda").to(dtype)
    out = block(x, positions, attention.offsets(lengths))
    out.backward(dout)
    xd = x.detach().double().requires_grad_(True)
    want, w = _plain(block, xd, positions, lengths, causal)
    want.backward(dout.double())
    assert _rms(out.double() - want) <= 8 * U[dtype] * _rms(want)
    assert _rms(x.grad.double() - xd.grad) <= 16 * U[dtype] * _rms(xd.grad)
    for name, p in block.named_parameters():
        assert _rms(p.grad.double() - w[name].grad) <= 16 * U[dtype] * _rms(w[name].grad), name


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_and_steps(cuda, dtype):
    """A prompt, then token by token over the cache: the rows of the causal pass over all."""
    from hi3d_amd import torso

    torch.manual_seed(1)
    block = torso.TokenAttention(256, 4, 2, axes=1, causal=True, dtype=dtype, device="cuda")
    x = torch.randn(90, 256, device="cuda").to(dtype)
    positions = torch.arange(90, device="cuda", dtype=torch.int32)[:, None]
    want = _plain(block, x.double(), positions, [90], True)[0].detach()
    cache = torso.KeyValueCache(1, 90, 2, 64, dtype)
    with torch.no_grad():
        rows = [block(x[:70], positions[:70], cache=cache)]
        for i in range(70, 90):
            rows.append(block.step(x[i:i + 1], positions[i:i + 1], cache))
    assert _rms(torch.cat(rows).double() - want) <= 8 * U[dtype] * _rms(want)
    assert cache.used == [90] and int(cache.lens[0]) == 90
    with pytest.raises(ValueError, match="no room"):
        block.step(x[:1], positions[:1], cache)


def test_steps_of_sequences_of_different_lengths(cuda):
    from hi3d_amd import torso

    torch.manual_seed(2)
    block = torso.TokenAttention(128, 2, axes=1, causal=True, device="cuda")
    lengths, room = [33, 1, 64], 70
    x = torch.randn(3, room, 128, device="cuda").half()
    positions = torch.arange(room, device="cuda", dtype=torch.int32)[:, None]
    cache = torso.KeyValueCache(3, room, 2, 64)
    with torch.no_grad():
        for b, n in enumerate(lengths):
            _, k, v = block.project(x[b, :n], positions[:n])
            cache.extend(b, k, v)
        got = block.step(torch.stack([x[b, n] for b, n in enumerate(lengths)]),
                         torch.tensor([[n] for n in lengths], device="cuda", dtype=torch.int32), cache)
    for b, n in enumerate(lengths):
        want = _plain(block, x[b, :n + 1].double(), positions[:n + 1], [n + 1], True)[0].detach()[-1]
        assert _rms(got[b].double() - want) <= 8 * U[torch.float16] * _rms(want)
