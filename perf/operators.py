"""The transformer torso's token operators at the sizes that programs call them with:
rotary positions, and attention over packed sequences of tokens, forward and backward.

``op`` of a case says which call it is:

* ``rotary``: queries and keys turned by their positions; with ``grad`` also the gradients
  of both.
* ``attend``: attention of packed sequences (every sequence attends to its own keys).
* ``query``: one new token of each sequence over a long cache of keys and values.
* ``grad``: attention and the gradients of queries, keys and values.

Rotary positions turn pair ``p`` of a token by ``sum_a position[a] * freqs[a, p]``; a voxel
token has three positions, each with its own third of the pairs. Attention is
``softmax(scale * q k^T) v`` with the query heads shared out over fewer key heads where
their numbers differ; a causal query ``i`` of ``Lq`` sees the keys ``j <= i + Lk - Lq``; a
row that sees no key gives zeros.

With ``own`` false everything is elementary torch operations in 32 bits (angles in 64).
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parent.parent / "hi3dv1.0-mlx_amd")

CHUNK = 1 << 27
"""Scores held at once by the plain form."""


# ---------------------------------------------------------------------------- cases


def listed() -> list[dict]:
    return [
        # Rotating one token of a served sequence far into its context: launch latency.
        dict(name="rotary_1x32x128_fp16", op="rotary", tokens=1, hq=32, hk=8, dim=128, rot=128, axes=1,
             layout="half", stretch=1.0, dtype="float16", grad=False),
        # The refiner's tokens (2112 channels as 33 heads of 64) by their voxel coordinates.
        dict(name="rotary_20011x33x64_fp16", op="rotary", tokens=20011, hq=33, hk=33, dim=64, rot=64, axes=3,
             layout="interleaved", stretch=1.0, dtype="float16", grad=False),
        # Training on long sequences: half of each head turns, positions stretched four times.
        dict(name="rotary_grad_65536x32x128_bf16", op="rotary", tokens=65536, hq=32, hk=8, dim=128, rot=64, axes=1,
             layout="half", stretch=4.0, dtype="bfloat16", grad=True),
        # A small object's tokens.
        dict(name="attend_517x8x64_fp16", op="attend", tokens_q=517, tokens_k=517, count=1, ragged=False, hq=8, hk=8,
             dim=64, causal=False, keep=1.0, dtype="float16"),
        # The decoder's windows of 48 serialized voxels on 327,581 voxels, 256 channels.
        dict(name="attend_windows_327581x8x32_fp16", op="attend", tokens_q=327581, tokens_k=327581, count=6825,
             ragged=False, hq=8, hk=8, dim=32, causal=False, keep=1.0, dtype="float16"),
        # Full attention over the tokens of two objects in a batch.
        dict(name="attend_20011x33x64_fp16", op="attend", tokens_q=20011, tokens_k=20011, count=2, ragged=True, hq=33,
             hk=33, dim=64, causal=False, keep=1.0, dtype="float16"),
        # Tokens of two objects over padded condition tokens, of which a part is masked.
        dict(name="cross_20011x2060x24x88_bf16", op="attend", tokens_q=20011, tokens_k=2060, count=2, ragged=True,
             hq=24, hk=24, dim=88, causal=False, keep=0.8, dtype="bfloat16"),
        # A long prompt, causal, four query heads to a key head.
        dict(name="causal_16384x32x8x128_bf16", op="attend", tokens_q=16384, tokens_k=16384, count=1, ragged=False,
             hq=32, hk=8, dim=128, causal=True, keep=1.0, dtype="bfloat16"),
        # One new token of each of eight sequences over long caches filled to different lengths.
        dict(name="query_8x65536x32x8x128_bf16", op="query", count=8, cache=65536, hq=32, hk=8, dim=128,
             dtype="bfloat16"),
        # One new token of one sequence over a short cache.
        dict(name="query_1x1030x33x64_fp16", op="query", count=1, cache=1030, hq=33, hk=33, dim=64, dtype="float16"),
        # A training step over the tokens of four objects of different sizes.
        dict(name="grad_8191x33x64_fp16", op="grad", tokens_q=8191, tokens_k=8191, count=4, ragged=True, hq=33, hk=33,
             dim=64, causal=False, keep=1.0, dtype="float16"),
        # A training step over two causal sequences with shared key heads.
        dict(name="grad_causal_8192x32x8x128_bf16", op="grad", tokens_q=8192, tokens_k=8192, count=2, ragged=False,
             hq=32, hk=8, dim=128, causal=True, keep=1.0, dtype="bfloat16"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    op = rng.choice(["rotary", "attend", "attend", "query", "grad", "grad"])
    dtype = rng.choice(["float16", "bfloat16"])
    hq, hk, dim = rng.choice([(33, 33, 64), (8, 8, 32), (24, 24, 88), (32, 8, 128), (16, 2, 96), (12, 1, 64),
                              (16, 16, 128)])
    if op == "rotary":
        dtype = rng.choice([dtype, "float32"])
        most = 65536 * 40 * 128 // ((hq + hk) * dim * (2 if dtype == "float32" else 1))
        return dict(op=op, tokens=_log_int(rng, 1, min(65536, most)), hq=hq, hk=hk, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2]), axes=rng.choice([1, 3]),
                    layout=rng.choice(["half", "interleaved"]), stretch=rng.choice([1.0, 4.0]), dtype=dtype,
                    grad=rng.random() < 0.5)
    if op == "query":
        count = rng.choice([1, 3, 8, 32])
        most = 8 * 65536 * 8 * 128 // (count * hk * dim)
        return dict(op=op, count=count, cache=_log_int(rng, 64, min(most, 131072)), hq=hq, hk=hk, dim=dim, dtype=dtype)
    causal, count = rng.random() < 0.4, rng.choice([1, 2, 5, 16])
    pairs = 10 ** rng.uniform(5.0, 8.3 if op == "grad" else 9.0) * (8 * 64) / (hq * max(dim, 64))
    across = 1.0 if causal else math.exp(rng.uniform(-0.7, 0.7))
    tokens_q = max(count, min(32768, int(math.sqrt(pairs * count) * across)))
    tokens_k = tokens_q if causal else max(count, min(32768, int(pairs * count / tokens_q)))
    return dict(op=op, tokens_q=tokens_q, tokens_k=tokens_k, count=count, ragged=rng.random() < 0.7, hq=hq, hk=hk,
                dim=dim, causal=causal, keep=rng.choice([1.0, 1.0, 0.8]), dtype=dtype)


def _lengths(total: int, count: int, ragged: bool) -> list[int]:
    """``count`` lengths that sum to ``total``: equal ones and a remainder, or uneven ones."""
    if not ragged:
        size = -(-total // count)
        return [max(0, min(size, total - i * size)) for i in range(count)]
    share = [1.0 + (i * 7919 + 6) % 10 / 5 for i in range(count)]
    ends = [round(total * sum(share[:i + 1]) / sum(share)) for i in range(count)]
    return [b - a for a, b in zip([0] + ends, ends)]


def _pairs(case: dict) -> float:
    """(query, key) pairs that a case's mask leaves, per head."""
    lq, lk = (_lengths(case[t], case["count"], case["ragged"]) for t in ("tokens_q", "tokens_k"))
    if not case["causal"]:
        return case["keep"] * sum(a * b for a, b in zip(lq, lk))
    return case["keep"] * sum(a * (a + 1) / 2 for a in lq)


# --------------------------------------------------------------------------- inputs


def _normal(shape, seed: int, i: int, dtype) -> torch.Tensor:
    g = torch.Generator(device="cuda").manual_seed(seed + 1_000_003 * i)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _offsets(lengths: list[int]) -> torch.Tensor:
    return torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0).int().cuda()


def _frequencies(case: dict) -> torch.Tensor:
    """``[axes, rot / 2]`` in 64 bits: powers of 1/10000, each axis on its own run of pairs
    (pairs that are left over stay as they are)."""
    axes, pairs = case["axes"], case["rot"] // 2
    each = pairs // axes
    f = torch.zeros(axes, pairs, dtype=torch.float64)
    power = 10000.0 ** (-torch.arange(each, dtype=torch.float64) / each) / case["stretch"]
    for a in range(axes):
        f[a, a * each:(a + 1) * each] = power
    return f.cuda()


def prepare(case: dict, seed: int) -> dict:
    op, dt = case["op"], getattr(torch, case["dtype"])
    hq, hk, d = case["hq"], case["hk"], case["dim"]
    s = {"case": case, "op": op}
    g = torch.Generator(device="cuda").manual_seed(seed)
    if op == "rotary":
        n = case["tokens"]
        qkv = _normal((n, hq + 2 * hk, d), seed, 1, dt)  # queries and keys as the joint projection leaves them
        s["q"], s["k"] = qkv[:, :hq], qkv[:, hq:hq + hk]
        if case["axes"] == 3:  # voxel rows (batch, x, y, z)
            s["positions"] = torch.randint(0, 512, (n, 4), generator=g, device="cuda", dtype=torch.int32)[:, 1:]
        else:
            start = int(torch.randint(0, 100_000, (1,), generator=g, device="cuda"))
            s["positions"] = torch.arange(start, start + n, device="cuda", dtype=torch.int32)[:, None]
        s["freqs"] = _frequencies(case)
        if case["grad"]:
            s["dq"], s["dk"] = _normal((n, hq, d), seed, 2, dt), _normal((n, hk, d), seed, 3, dt)
            s["q"].requires_grad_(True), s["k"].requires_grad_(True)
        return s
    if op == "query":
        b, cache = case["count"], case["cache"]
        s["q"] = _normal((b, 1, hq, d), seed, 1, dt)
        s["k"], s["v"] = _normal((b, cache, hk, d), seed, 2, dt), _normal((b, cache, hk, d), seed, 3, dt)
        lens = torch.randint(max(1, cache * 3 // 4), cache + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        s["lens"] = lens
        return s
    nq, nk = case["tokens_q"], case["tokens_k"]
    lq, lk = _lengths(nq, case["count"], case["ragged"]), _lengths(nk, case["count"], case["ragged"])
    s["lengths"], s["cu_q"], s["cu_k"] = list(zip(lq, lk)), _offsets(lq), _offsets(lk)
    if nq == nk:  # views of one projection
        qkv = _normal((nq, hq + 2 * hk, d), seed, 1, dt)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    else:
        kv = _normal((nk, 2, hk, d), seed, 2, dt)
        s["q"], s["k"], s["v"] = _normal((nq, hq, d), seed, 1, dt), kv[:, 0], kv[:, 1]
    s["mask"] = None
    if case["keep"] < 1:
        s["mask"] = torch.rand(nk, generator=g, device="cuda") < case["keep"]
    if op == "grad":
        s["dout"] = _normal((nq, hq, d), seed, 4, dt)
        s["q"], s["k"], s["v"] = (s[t].detach().requires_grad_(True) for t in "qkv")
    return s


# ------------------------------------------------------------------------ the calls


def run(s: dict):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s: dict):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from hi3d_amd import attention, rotary

    case, op = s["case"], s["op"]
    if op == "rotary":
        q, k = rotary.rotate_qk(s["q"], s["k"], s["positions"], s["freqs"], layout=case["layout"])
        if not case["grad"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    if op == "query":
        return attention.attend(s["q"], s["k"], s["v"], lens_k=s["lens"])
    out = attention.attend(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=case["causal"], key_mask=s["mask"])
    if op == "attend":
        return out
    dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


@torch.no_grad()
def _run_plain(s: dict):
    case, op = s["case"], s["op"]
    if op == "rotary":
        angle = s["positions"].double() @ s["freqs"]
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
        turn = lambda x, to: _turn(x, cos, to * sin, case["rot"], case["layout"])  # noqa: E731
        out = {"q": turn(s["q"], 1.0), "k": turn(s["k"], 1.0)}
        if case["grad"]:
            out |= {"dq": turn(s["dq"], -1.0), "dk": turn(s["dk"], -1.0)}
        return out
    if op == "query":
        dark = torch.arange(case["cache"], device="cuda") >= s["lens"][:, None]
        return _plain_attend(s["q"], s["k"], s["v"], dark[:, None, None, None, :]).to(s["q"].dtype)
    grad = op == "grad"
    out = {"out": torch.empty_like(s["q"], memory_format=torch.contiguous_format)}
    if grad:
        out |= {"d" + t: torch.empty_like(s[t], memory_format=torch.contiguous_format) for t in "qkv"}
    at_q = at_k = 0
    run_of = 1
    for i in range(0, len(s["lengths"])):
        lq, lk = s["lengths"][i]
        if i + 1 < len(s["lengths"]) and s["lengths"][i + 1] == (lq, lk) and run_of * lq * lk * case["hq"] < CHUNK:
            run_of += 1  # neighbours of the same lengths are one batch
            continue
        rq, rk = slice(at_q, at_q + run_of * lq), slice(at_k, at_k + run_of * lk)
        at_q, at_k = rq.stop, rk.stop
        _plain_sequences(s, out, rq, rk, run_of, lq, lk, grad)
        run_of = 1
    return out if grad else out["out"]


def _turn(x, cos, sin, rot, layout):
    y = x.float()
    turned, rest = y[..., :rot], y[..., rot:]
    if layout == "half":
        a, b = turned.chunk(2, -1)
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, rest], -1).to(x.dtype)


def _plain_sequences(s, out, rq, rk, count, lq, lk, grad):
    """``count`` sequences of ``lq`` queries and ``lk`` keys each, a chunk of key heads at a time."""
    case = s["case"]
    dark = None
    if case["causal"]:
        dark = (torch.arange(lk, device="cuda") > torch.arange(lq, device="cuda")[:, None] + (lk - lq))[None, None, None]
    if s["mask"] is not None:
        hidden = ~s["mask"][rk].reshape(count, 1, 1, 1, lk)
        dark = hidden if dark is None else dark | hidden
    group = case["hq"] // case["hk"]
    step = max(1, CHUNK // max(1, count * lq * lk * group))
    for h in range(0, case["hk"], step):
        hk, hq = slice(h, min(h + step, case["hk"])), slice(h * group, min(h + step, case["hk"]) * group)
        q = s["q"][rq, hq].reshape(count, lq, -1, case["dim"])
        k, v = (s[t][rk, hk].reshape(count, lk, -1, case["dim"]) for t in "kv")
        if not grad:
            out["out"][rq, hq] = _plain_attend(q, k, v, dark).flatten(0, 1).to(q.dtype)
            continue
        dout = s["dout"][rq, hq].reshape(count, lq, -1, case["dim"])
        for name, value in zip(("out", "dq", "dk", "dv"), _plain_grad(q, k, v, dout, dark)):
            out[name][(rk, hk) if name in ("dk", "dv") else (rq, hq)] = value.flatten(0, 1).to(q.dtype)


def _by_head(x, heads):
    """``[B, L, H, D]`` as ``[B, heads, H / heads, L, D]`` in 32 bits."""
    b, n, h, d = x.shape
    return x.float().reshape(b, n, heads, h // heads, d).permute(0, 2, 3, 1, 4)


def _by_token(x):
    return x.permute(0, 3, 1, 2, 4).flatten(2, 3)


def _probabilities(q, k, dark):
    score = (q * q.shape[-1] ** -0.5) @ k.transpose(-1, -2)
    if dark is None:
        top = score.amax(-1, keepdim=True)
    else:
        score = score.masked_fill_(dark, -math.inf)
        top = score.amax(-1, keepdim=True).clamp_(min=-3e38)  # a row that sees no key
    p = (score - top).exp_()
    return p / p.sum(-1, keepdim=True).clamp_(min=1e-38)


def _plain_attend(q, k, v, dark):
    heads = k.shape[2]
    q, k, v = (_by_head(x, heads) for x in (q, k, v))
    if not k.shape[-2]:
        return _by_token(torch.zeros_like(q))
    return _by_token(_probabilities(q, k, dark) @ v)


def _plain_grad(q, k, v, dout, dark):
    heads = k.shape[2]
    q, k, v, dout = (_by_head(x, heads) for x in (q, k, v, dout))
    scale = q.shape[-1] ** -0.5
    if not k.shape[-2]:
        return _by_token(torch.zeros_like(q)), _by_token(torch.zeros_like(q)), _by_token(k), _by_token(v)
    p = _probabilities(q, k, dark)
    out = p @ v
    dv = (p.transpose(-1, -2) @ dout).sum(2, keepdim=True)
    ds = p * (dout @ v.transpose(-1, -2) - (dout * out).sum(-1, keepdim=True))
    dq = ds @ k * scale
    dk = (ds.transpose(-1, -2) @ q).sum(2, keepdim=True) * scale
    return _by_token(out), _by_token(dq), _by_token(dk), _by_token(dv)


# ------------------------------------------------------------------- work, 64 bits


def work(case: dict) -> dict:
    hq, hk, d, e = case["hq"], case["hk"], case["dim"], 4 if case["dtype"] == "float32" else 2
    if case["op"] == "rotary":
        n, passes = case["tokens"], 2 if case["grad"] else 1
        values = n * (hq + hk) * d
        return {"bytes": passes * 2 * e * values + 4 * n * case["axes"], "flops": passes * 3 * n * (hq + hk) * case["rot"]}
    if case["op"] == "query":
        keys = case["count"] * case["cache"] * 7 / 8
        return {"bytes": e * (2 * keys * hk * d + 2 * case["count"] * hq * d), "flops": 4 * keys * hq * d}
    q, k = case["tokens_q"] * hq * d, case["tokens_k"] * hk * d
    if case["op"] == "attend":
        return {"bytes": e * (2 * q + 2 * k), "flops": 4 * _pairs(case) * hq * d}
    return {"bytes": e * (4 * q + 4 * k), "flops": 14 * _pairs(case) * hq * d}


@torch.no_grad()
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        angle = sum(s["positions"][:, a].double()[:, None] * s["freqs"][a] for a in range(case["axes"]))
        wave, rot = torch.polar(torch.ones_like(angle), angle)[:, None], case["rot"]

        def turned(x, w):
            x = x.double()
            y, half = x.clone(), rot // 2
            first, second = (slice(0, half), slice(half, rot)) if case["layout"] == "half" else (slice(0, rot, 2), slice(1, rot, 2))
            z = torch.complex(x[..., first], x[..., second]) * w
            y[..., first], y[..., second] = z.real, z.imag
            return y

        out = {"q": turned(s["q"], wave), "k": turned(s["k"], wave)}
        return out | ({"dq": turned(s["dq"], wave.conj()), "dk": turned(s["dk"], wave.conj())} if case["grad"] else {})
    hq, hk, d = case["hq"], case["hk"], case["dim"]
    group, scale = hq // hk, 1 / math.sqrt(d)
    if case["op"] == "query":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lens"].tolist()):
            for h in range(hk):
                k, v = s["k"][b, :n, h].double(), s["v"][b, :n, h].double()
                for g in range(h * group, (h + 1) * group):
                    out[b, 0, g] = torch.softmax(scale * (k @ s["q"][b, 0, g].double()), 0) @ v
        return out
    grad = case["op"] == "grad"
    out = {t: torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda") for t in (("out", "dq") if grad else ("out",))}
    if grad:
        out |= {t: torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda") for t in ("dk", "dv")}
    q0 = k0 = 0
    for lq, lk in s["lengths"]:
        q1, k1 = q0 + lq, k0 + lk
        seen = torch.ones(lq, lk, dtype=torch.bool, device="cuda")
        if case["causal"]:
            seen = seen.tril(lk - lq)
        if s["mask"] is not None:
            seen = seen & s["mask"][k0:k1]
        some = max(1, (1 << 26) // max(1, lq * lk))
        for g in range(0, hq, some) if lq and lk else ():
            heads = torch.arange(g, min(g + some, hq), device="cuda")
            of = heads // group
            q, k, v = s["q"][q0:q1, heads].double().movedim(1, 0), *(s[t][k0:k1, of].double().movedim(1, 0) for t in "kv")
            score = torch.where(seen, scale * torch.bmm(q, k.mT.contiguous()), -math.inf)
            p = torch.softmax(score, -1).nan_to_num_(0.0)
            o = torch.bmm(p, v)
            out["out"][q0:q1, heads] = o.movedim(0, 1)
            if grad:
                do = s["dout"][q0:q1, heads].double().movedim(1, 0)
                ds = p * (torch.bmm(do, v.mT.contiguous()) - (do * o).sum(-1, keepdim=True)) * scale
                out["dq"][q0:q1, heads] = torch.bmm(ds, k).movedim(0, 1)
                out["dk"][k0:k1].index_add_(1, of, torch.bmm(ds.mT.contiguous(), q).movedim(0, 1))
                out["dv"][k0:k1].index_add_(1, of, torch.bmm(p.mT.contiguous(), do).movedim(0, 1))
        q0, k0 = q1, k1
    return out if grad else out["out"]
