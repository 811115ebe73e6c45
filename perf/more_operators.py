"""Attention whose scores carry more than the product of a query and a key, at the sizes that
programs call it with: forward, backward and single tokens over a cache.

``op`` of a case says which call it is:

* ``attend``: packed sequences, every one over its own keys;
* ``grad``: the same and the gradients of queries, keys and values (and of the learned bias);
* ``query``: one new token of each sequence over a cache of keys and values;
* ``shared``: new tokens of each sequence over keys that all sequences share (a long common
  beginning) and then over a cache of its own.

What the scores carry, for query ``i`` of ``lq`` at place ``i + lk - lq`` among ``lk`` keys and key
``j``, with ``r = j - (i + lk - lq)``:

* ``cap``: ``s = cap * tanh(scale q k / cap)`` in place of ``s = scale q k`` (0: none);
* ``slopes``: ``s - slope[head] * |r|``;
* ``buckets``: ``s + bias[bucket[clamp(r, -far, far)], head]`` with a learned table;
* ``prefix``: a causal sequence whose first keys are seen by all of its queries.

Key heads are shared by groups of query heads where their numbers differ; a row that sees no
key gives zeros. With ``own`` false everything is elementary torch operations in 32 bits.
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


def _packed(name, op, tokens, count, ragged, hq, hk, dim, dtype, causal=False, cap=0.0, slopes=False, buckets=0, far=0,
            prefix=0.0) -> dict:
    case = dict(op=op, tokens=tokens, count=count, ragged=ragged, hq=hq, hk=hk, dim=dim, dtype=dtype, causal=causal,
                cap=cap, slopes=slopes, buckets=buckets, far=far, prefix=prefix)
    return dict(name=name, **case) if name else case


def _cached(name, op, count, new, cache, shared, hq, hk, dim, dtype, cap=0.0, slopes=False, buckets=0, far=0) -> dict:
    case = dict(op=op, count=count, new=new, cache=cache, shared=shared, hq=hq, hk=hk, dim=dim, dtype=dtype, cap=cap,
                slopes=slopes, buckets=buckets, far=far)
    return dict(name=name, **case) if name else case


def listed() -> list[dict]:
    return [
        # One new token over a short cache, capped scores: launch latency.
        _cached("cap_query_1x1030x16x2x128_bf16", "query", 1, 1, 1030, 0, 16, 2, 128, "bfloat16", cap=50.0),
        # One new token of each of eight sequences over long caches, distances by slopes.
        _cached("slopes_query_8x32768x32x8x128_bf16", "query", 8, 1, 32768, 0, 32, 8, 128, "bfloat16", slopes=True),
        # Prompts whose condition tokens are seen by all that follows, capped scores.
        _packed("prefix_cap_8191x32x8x128_bf16", "attend", 8191, 3, True, 32, 8, 128, "bfloat16", True, 30.0, prefix=0.3),
        # The refiner's tokens (33 heads of 64) of two objects in their serialized order, nearer ones first.
        _packed("slopes_20011x33x64_fp16", "attend", 20011, 2, True, 33, 33, 64, "float16", slopes=True),
        # A training step over two prompts with seen prefixes, capped scores, shared key heads.
        _packed("grad_prefix_cap_8192x32x8x128_bf16", "grad", 8192, 2, False, 32, 8, 128, "bfloat16", True, 50.0, prefix=0.25),
        # A training step over objects of different sizes, nearer tokens first.
        _packed("grad_slopes_4099x16x64_fp16", "grad", 4099, 3, True, 16, 16, 64, "float16", slopes=True),
        # The decoder's windows of 48 serialized voxels, 256 channels, with a learned bias.
        _packed("bias_windows_327581x8x32_fp16", "attend", 327581, 6825, False, 8, 8, 32, "float16", buckets=32, far=128),
        # A long prompt, causal, with a learned bias that is flat past 128 tokens.
        _packed("bias_causal_12289x32x8x128_bf16", "attend", 12289, 1, False, 32, 8, 128, "bfloat16", True, buckets=32,
                far=128),
        # A training step with a learned bias over the tokens of four objects.
        _packed("bias_grad_8191x33x64_fp16", "grad", 8191, 4, True, 33, 33, 64, "float16", buckets=32, far=128),
        # The smallest training step that fills no more than a part of the chip.
        _packed("bias_grad_517x8x64_bf16", "grad", 517, 1, False, 8, 8, 64, "bfloat16", buckets=32, far=128),
        # Thirty-two answers to one long prompt, a token each.
        _cached("shared_32x16384+700x32x8x128_bf16", "shared", 32, 1, 700, 16384, 32, 8, 128, "bfloat16"),
        # Four sequences after a short common beginning, drafts of three tokens each, capped scores.
        _cached("shared_4x3x1030+77x33x64_fp16", "shared", 4, 3, 77, 1030, 33, 33, 64, "float16", cap=50.0),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    op = rng.choice(["attend", "attend", "grad", "grad", "query", "shared", "shared"])
    dtype = rng.choice(["float16", "bfloat16"])
    hq, hk, dim = rng.choice([(33, 33, 64), (8, 8, 32), (24, 24, 88), (32, 8, 128), (16, 2, 96), (12, 1, 64),
                              (16, 16, 128)])
    kind = rng.choice(["cap", "slopes", "buckets", "buckets", "cap and slopes", "cap and buckets"])
    terms = dict(cap=rng.choice([20.0, 50.0]) if "cap" in kind else 0.0, slopes="slopes" in kind,
                 buckets=rng.choice([16, 32, 64]) if "buckets" in kind else 0, far=rng.choice([48, 128, 400]))
    terms["far"] *= terms["buckets"] > 0
    if op in ("query", "shared"):
        count = rng.choice([1, 3, 8, 32]) if op == "query" else rng.choice([2, 5, 16, 48])
        new = 1 if op == "query" else rng.choice([1, 1, 4])
        keys = 8 * 32768 * 8 * 128 // (hk * dim)  # of the largest listed case
        if op == "query":
            return _cached("", op, count, new, _log_int(rng, 64, min(keys // count, 65536)), 0, hq, hk, dim, dtype, **terms)
        return _cached("", op, count, new, _log_int(rng, 16, min(keys // count // 2, 2048)), _log_int(rng, 64, 16384), hq, hk,
                       dim, dtype, **terms)
    causal, count = rng.random() < 0.5, rng.choice([1, 2, 5, 16])
    pairs = 10 ** rng.uniform(5.0, 7.8 if op == "grad" else 8.3) * (8 * 64) / (hq * max(dim, 64))
    tokens = max(count, min(16384, int(math.sqrt(pairs * count))))
    return _packed("", op, tokens, count, rng.random() < 0.7, hq, hk, dim, dtype, causal,
                   prefix=rng.choice([0.0, 0.4]) if causal else 0.0, **terms)


def _lengths(total: int, count: int, ragged: bool) -> list[int]:
    """``count`` lengths that sum to ``total``: equal ones and a remainder, or uneven ones."""
    if not ragged:
        size = -(-total // count)
        return [max(0, min(size, total - i * size)) for i in range(count)]
    share = [1.0 + (i * 7919 + 6) % 10 / 5 for i in range(count)]
    ends = [round(total * sum(share[:i + 1]) / sum(share)) for i in range(count)]
    return [b - a for a, b in zip([0] + ends, ends)]


def _prefixes(case: dict) -> list[int]:
    """How many first keys of each sequence all of its queries see."""
    return [round(n * case["prefix"] * (0.5 + (i * 3 + 1) % 4 / 4)) for i, n in
            enumerate(_lengths(case["tokens"], case["count"], case["ragged"]))]


def _pairs(case: dict) -> float:
    """(query, key) pairs that a packed case's queries see, per head."""
    lengths = _lengths(case["tokens"], case["count"], case["ragged"])
    if not case["causal"]:
        return sum(n * n for n in lengths)
    return sum(n * (n + 1) / 2 + p * (p - 1) / 2 for n, p in zip(lengths, _prefixes(case)))


# --------------------------------------------------------------------------- inputs


def _normal(shape, seed: int, i: int, dtype) -> torch.Tensor:
    g = torch.Generator(device="cuda").manual_seed(seed + 1_000_003 * i)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _bucket_map(count: int, far: int, causal: bool) -> torch.Tensor:
    """``[2 far + 1]``: the bucket of each relative position ``-far .. far``. Half of the buckets
    for each side (all of them for the keys before, where the later ones are not seen); in a side
    the first half holds a distance each, the others distances that grow by a constant factor up
    to ``far``."""
    side = count if causal else count // 2
    near = side // 2
    rest = side - near

    def place(d: int) -> int:
        if d < near:
            return d
        n = 0  # the largest with d >= near (far / near) ** (n / rest), in whole numbers
        while n + 1 < rest and d ** rest * near ** (n + 1) >= far ** (n + 1) * near ** rest:
            n += 1
        return near + n

    before = [place(d) for d in range(far, 0, -1)]
    after = [0 if causal else side + place(d) for d in range(1, far + 1)]
    return torch.tensor(before + [0] + after, dtype=torch.int32)


def prepare(case: dict, seed: int) -> dict:
    op, dt = case["op"], getattr(torch, case["dtype"])
    hq, hk, d = case["hq"], case["hk"], case["dim"]
    s = {"case": case, "cap": case["cap"] or None, "slopes": None, "bias": None, "buckets": None}
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["slopes"]:
        s["slopes"] = (2.0 ** (-8.0 * torch.arange(1, hq + 1) / hq)).float().cuda()
    if case["buckets"]:
        s["bias"] = _normal((case["buckets"], hq), seed, 5, dt)
        s["buckets"] = _bucket_map(case["buckets"], case["far"], case.get("causal", True)).cuda()
    gain = 4.0 if case["cap"] else 1.0  # scores that reach the cap's bend
    if op in ("query", "shared"):
        b, new, cache = case["count"], case["new"], case["cache"]
        s["q"] = _normal((b, new, hq, d), seed, 1, torch.float32).mul_(gain).to(dt)
        s["k"], s["v"] = _normal((b, cache, hk, d), seed, 2, dt), _normal((b, cache, hk, d), seed, 3, dt)
        s["lens"] = torch.randint(max(new, cache // 2), cache + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        if op == "shared":
            s["pk"], s["pv"] = _normal((case["shared"], hk, d), seed, 6, dt), _normal((case["shared"], hk, d), seed, 7, dt)
        return s
    n = case["tokens"]
    s["lengths"] = _lengths(n, case["count"], case["ragged"])
    s["cu"] = torch.tensor([0] + s["lengths"], dtype=torch.int32).cumsum(0).int().cuda()
    s["prefixes"] = _prefixes(case)
    s["prefix"] = torch.tensor(s["prefixes"], dtype=torch.int32).cuda() if case["prefix"] else None
    qkv = _normal((n, hq + 2 * hk, d), seed, 1, torch.float32)  # one projection's output
    qkv[:, :hq] *= gain
    qkv = qkv.to(dt)
    s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    if op == "grad":
        s["dout"] = _normal((n, hq, d), seed, 4, dt)
        s["q"], s["k"], s["v"] = (s[t].detach().requires_grad_(True) for t in "qkv")
        if s["bias"] is not None:
            s["bias"].requires_grad_(True)
    return s


# ------------------------------------------------------------------------ the calls


def run(s: dict):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s: dict):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from hi3d_amd import attention

    case = s["case"]
    terms = dict(cap=s["cap"], slopes=s["slopes"], bias=s["bias"], buckets=s["buckets"])
    if case["op"] == "query":
        return attention.attend(s["q"], s["k"], s["v"], lens_k=s["lens"], **terms)
    if case["op"] == "shared":
        return attention.attend_shared(s["q"], s["pk"], s["pv"], s["k"], s["v"], lens_k=s["lens"], causal=True, **terms)
    out = attention.attend(s["q"], s["k"], s["v"], s["cu"], causal=case["causal"], prefix=s["prefix"], **terms)
    if case["op"] == "attend":
        return out
    names = ["q", "k", "v"] + ["bias"] * (s["bias"] is not None)
    grads = torch.autograd.grad(out, [s[t] for t in names], s["dout"])
    return {"out": out.detach(), **{"d" + t: x for t, x in zip(names, grads)}}


@torch.no_grad()
def _run_plain(s: dict):
    case = s["case"]
    if case["op"] in ("query", "shared"):
        return _plain_cached(s)
    grad = case["op"] == "grad"
    out = {"out": torch.empty_like(s["q"], memory_format=torch.contiguous_format)}
    if grad:
        out |= {"d" + t: torch.empty_like(s[t], memory_format=torch.contiguous_format) for t in "qkv"}
    dbias = torch.zeros(case["buckets"], case["hq"], dtype=torch.float64, device="cuda")
    at, run_of, lengths = 0, 1, list(zip(s["lengths"], s["prefixes"]))
    for i, (n, prefix) in enumerate(lengths):
        if i + 1 < len(lengths) and lengths[i + 1] == (n, prefix) and run_of * n * n * case["hq"] < CHUNK:
            run_of += 1  # neighbours of the same lengths are one batch
            continue
        _plain_sequences(s, out, dbias, slice(at, at + run_of * n), run_of, n, prefix, grad)
        at += run_of * n
        run_of = 1
    if not grad:
        return out["out"]
    return out | ({"dbias": dbias.to(s["bias"].dtype)} if case["buckets"] else {})


def _plain_sequences(s, out, dbias, rows, count, n, prefix, grad):
    """``count`` sequences of ``n`` tokens each, some key heads at a time."""
    case = s["case"]
    r = torch.arange(n, device="cuda") - torch.arange(n, device="cuda")[:, None]
    dark = None
    if case["causal"]:
        dark = (r > 0) & (torch.arange(n, device="cuda") >= prefix)
    group = case["hq"] // case["hk"]
    step = max(1, CHUNK // max(1, count * n * n * group))
    for h in range(0, case["hk"], step):
        hk, hq = slice(h, min(h + step, case["hk"])), slice(h * group, min(h + step, case["hk"]) * group)
        q = s["q"][rows, hq].reshape(count, n, -1, case["dim"])
        k, v = (s[t][rows, hk].reshape(count, n, -1, case["dim"]) for t in "kv")
        dout = s["dout"][rows, hq].reshape(count, n, -1, case["dim"]) if grad else None
        got = _plain(s, hq, q, k, v, r[None], dark, dout)
        for name, value in zip(("out", "dq", "dk", "dv"), got):
            out[name][rows, hk if name in ("dk", "dv") else hq] = value.flatten(0, 1).to(q.dtype)
        if grad and case["buckets"]:
            far, side = case["far"], torch.arange(1 - n, n, device="cuda")
            dbias[:, hq].index_add_(0, s["buckets"].long()[side.clamp(-far, far) + far], _diagonals(got[4]).T)


def _diagonals(x):
    """Sums of ``x [heads, n, n]`` over equal column - row, ``[heads, 2 n - 1]`` in 64 bits: rows from
    the last one on, each moved one place further."""
    heads, n, _ = x.shape
    x = torch.nn.functional.pad(x.flip(1), (0, n)).flatten(1)[:, :n * (2 * n - 1)]
    return x.reshape(heads, n, 2 * n - 1).sum(1, dtype=torch.float64)


def _plain_cached(s):
    """New tokens over the keys of a cache, behind those that all sequences share, if any."""
    case = s["case"]
    b, new = case["count"], case["new"]
    keys = torch.arange(-case["shared"], case["cache"], device="cuda")
    at = s["lens"][:, None] - new + torch.arange(new, device="cuda")  # place of each new token
    r = keys - at[:, :, None]
    k, v = s["k"], s["v"]
    if case["op"] == "shared":
        k, v = (torch.cat([s["p" + t].expand(b, -1, -1, -1), s[t]], 1) for t in "kv")
    group = case["hq"] // case["hk"]
    step = max(1, CHUNK // (b * new * keys.numel() * group))
    out = torch.empty_like(s["q"])
    for h in range(0, case["hk"], step):
        hk, hq = slice(h, min(h + step, case["hk"])), slice(h * group, min(h + step, case["hk"]) * group)
        out[:, :, hq] = _plain(s, hq, s["q"][:, :, hq], k[:, :, hk], v[:, :, hk], r, r[:, None, None] > 0, None)[0].to(out.dtype)
    return out


def _by_head(x, heads):
    """``[B, L, H, D]`` as ``[B, heads, H / heads, L, D]`` in 32 bits."""
    b, n, h, d = x.shape
    return x.float().reshape(b, n, heads, h // heads, d).permute(0, 2, 3, 1, 4)


def _by_token(x):
    return x.permute(0, 3, 1, 2, 4).flatten(2, 3)


def _plain(s, hq, q, k, v, r, dark, dout):
    """Output, and with ``dout`` the gradients of q, k and v and the scores' summed over sequences
    ``[heads, Lq, Lk]``. ``r [B or 1, Lq, Lk]``: relative positions."""
    case, heads = s["case"], k.shape[2]
    scale = case["dim"] ** -0.5
    group = q.shape[2] // heads
    q, k, v = (_by_head(x, heads) for x in (q, k, v))
    if not k.shape[-2]:
        return [_by_token(x) for x in ([q] if dout is None else [q, q, k, v])] + [q.new_zeros(heads * group, q.shape[-2], 0)]
    score = (q * scale) @ k.transpose(-1, -2)
    bend = None
    if case["cap"]:
        bend = score.div_(case["cap"]).tanh_()
        score = bend * case["cap"]
        bend = None if dout is None else bend
    if case["slopes"]:
        score -= s["slopes"][hq].reshape(1, heads, group, 1, 1) * r.abs().float()[:, None, None]
    if case["buckets"]:
        place = s["buckets"].long()[r.clamp(-case["far"], case["far"]) + case["far"]]
        table = s["bias"][:, hq].float().T.contiguous()
        score += table[:, place].reshape(heads, group, *place.shape).permute(2, 0, 1, 3, 4)
    if dark is not None:
        score.masked_fill_(dark, -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    p /= p.sum(-1, keepdim=True).clamp_(min=1e-38)
    out = p @ v
    if dout is None:
        return [_by_token(out)]
    dout = _by_head(dout, heads)
    dv = (p.transpose(-1, -2) @ dout).sum(2, keepdim=True)
    ds = p * (dout @ v.transpose(-1, -2) - (dout * out).sum(-1, keepdim=True))
    total = ds.sum(0).flatten(0, 1)
    if bend is not None:
        ds *= 1 - bend * bend
    dq = ds @ k * scale
    dk = (ds.transpose(-1, -2) @ q).sum(2, keepdim=True) * scale
    return [*map(_by_token, (out, dq, dk, dv)), total]


# ------------------------------------------------------------------- work, 64 bits


def work(case: dict) -> dict:
    hq, hk, d = case["hq"], case["hk"], case["dim"]
    table = 2 * case["buckets"] * hq
    if case["op"] in ("query", "shared"):
        own_keys = case["count"] * max(case["new"], case["cache"] * 3 / 4)
        rows = case["count"] * case["new"] * hq * d
        pairs = case["new"] * (own_keys + case["count"] * case["shared"])
        return {"bytes": 2 * (2 * (own_keys + case["shared"]) * hk * d + 2 * rows) + table, "flops": 4 * pairs * hq * d}
    q, k = case["tokens"] * hq * d, case["tokens"] * hk * d
    if case["op"] == "attend":
        return {"bytes": 2 * (2 * q + 2 * k) + table, "flops": 4 * _pairs(case) * hq * d}
    return {"bytes": 2 * (4 * q + 4 * k) + 2 * table, "flops": 14 * _pairs(case) * hq * d}


@torch.no_grad()
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    s["map"] = s["buckets"].tolist() if case["buckets"] else None
    group = case["hq"] // case["hk"]

    def scores(q, k, r, seen, head):
        """Scores ``[lq, lk]`` of one query head in 64 bits, and the derivative of the cap."""
        x, slope = torch.mm(q, k.mT.contiguous()) / math.sqrt(case["dim"]), 1.0
        if case["cap"]:
            w = torch.exp(-2 * x.abs() / case["cap"])
            x, slope = x.sign() * case["cap"] * (1 - w) / (1 + w), 4 * w / (1 + w) ** 2
        if s["slopes"] is not None:
            x = x - s["slopes"][head].double() * r.abs()
        if s["bias"] is not None:
            near = torch.minimum(torch.maximum(r, torch.full_like(r, -case["far"])), torch.full_like(r, case["far"]))
            x = x + s["bias"][:, head].double()[s["buckets"][near + case["far"]].long()]
        return torch.where(seen, x, -math.inf), slope

    if case["op"] in ("query", "shared"):
        out, new = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), case["new"]
        for b, n in enumerate(s["lens"].tolist()):
            r = torch.arange(-case["shared"], n, device="cuda") - torch.arange(n - new, n, device="cuda")[:, None]
            for h in range(case["hk"]):
                k, v = (s[t][b, :n, h].double() for t in "kv")
                if case["op"] == "shared":
                    k, v = torch.cat([s["pk"][:, h].double(), k]), torch.cat([s["pv"][:, h].double(), v])
                for g in range(h * group, (h + 1) * group):
                    x, _ = scores(s["q"][b, :, g].double(), k, r, r <= 0, g)
                    out[b, :, g] = torch.softmax(x, -1) @ v
        return out
    grad = case["op"] == "grad"
    if sum(n > 0 for n in s["lengths"]) > 200:  # windows: one batch of equal ones, and the last
        return _exact_windows(s)
    out = {t: torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda") for t in (("out", "dq") if grad else ("out",))}
    if grad:
        out |= {t: torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda") for t in ("dk", "dv")}
        if case["buckets"]:
            out["dbias"] = torch.zeros(s["bias"].shape, dtype=torch.float64, device="cuda")
    begin = 0
    for n, prefix in zip(s["lengths"], s["prefixes"]):
        end = begin + n
        place = torch.arange(n, device="cuda")
        r = place - place[:, None]
        seen = (r <= 0) | (place < prefix) if case["causal"] else torch.ones_like(r, dtype=torch.bool)
        all_ds = torch.zeros((case["hq"] if grad and case["buckets"] else 0), n, n, dtype=torch.float64, device="cuda")
        for head in range(case["hq"]) if n else ():
            q, k, v = s["q"][begin:end, head].double(), *(s[t][begin:end, head // group].double() for t in "kv")
            x, slope = scores(q, k, r, seen, head)
            p = torch.softmax(x, -1)
            o = p @ v
            out["out"][begin:end, head] = o
            if grad:
                do = s["dout"][begin:end, head].double()
                ds = p * (torch.mm(do, v.mT.contiguous()) - (do * o).sum(-1, keepdim=True))
                if case["buckets"]:
                    all_ds[head] = ds
                ds = ds * slope / math.sqrt(case["dim"])
                out["dq"][begin:end, head] = torch.mm(ds, k)
                out["dk"][begin:end, head // group] += torch.mm(ds.mT.contiguous(), q)
                out["dv"][begin:end, head // group] += torch.mm(p.mT.contiguous(), do)
        for side in range(1 - n, n) if len(all_ds) else ():
            bucket = s["map"][min(max(side, -case["far"]), case["far"]) + case["far"]]
            out["dbias"][bucket] += all_ds.diagonal(side, 1, 2).sum(-1)
        begin = end
    return out if grad else out["out"]


def _exact_windows(s: dict):
    """Many short sequences without a causal limit, forward: those of one length together."""
    case, out, begin = s["case"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    group, lengths = case["hq"] // case["hk"], s["lengths"]
    while begin < case["tokens"]:
        n = lengths[0]
        count = next((i for i, m in enumerate(lengths) if m != n), len(lengths))
        lengths, end = lengths[count:], begin + count * n
        place = torch.arange(n, device="cuda")
        r = (place - place[:, None]).clamp(-case["far"], case["far"])
        for head in range(case["hq"]):
            q, k, v = s["q"][begin:end, head], s["k"][begin:end, head // group], s["v"][begin:end, head // group]
            q, k, v = (x.double().reshape(count, n, case["dim"]) for x in (q, k, v))
            x = torch.bmm(q, k.mT.contiguous()) / math.sqrt(case["dim"])
            x = x + s["bias"][:, head].double()[s["buckets"][r + case["far"]].long()]
            out[begin:end, head] = torch.bmm(torch.softmax(x, -1), v).reshape(-1, case["dim"])
        begin = end
    return out
