"""What the tests of attention with terms share: problems, and checks against float64 with the
bounds of ``oracle.attention_terms``. The output is rounded once (half a step ``u`` of the type)
after probabilities that were rounded once for their product (``u``, and in fp16 2^-25 below its
normal range); gradients as there, products of two relative errors below 1 %."""

from __future__ import annotations

import numpy as np
import torch

from oracle import attention_terms as oterms

E = 2.0 ** -24
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}
DTYPES = [torch.float16, torch.bfloat16]


def host(x):
    return None if x is None else x.detach().double().cpu().numpy()


def ends(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)


def tensors(nq, nk, hq, hk, d, dtype, seed=0, gain=1.0):
    """q (times ``gain``), k, v and dout."""
    g = torch.Generator().manual_seed(seed)
    make = lambda n, h, s: (s * torch.randn((n, h, d), generator=g)).to(dtype).cuda()  # noqa: E731
    return make(nq, hq, gain), make(nk, hk, 1.0), make(nk, hk, 1.0), make(nq, hq, 1.0)


def terms(kind: str, heads: int, segments: int = 1, far: int = 9, count: int = 8, causal: bool = False, dtype=torch.float32,
          seed: int = 3, longest: int = 100):
    """Keyword arguments of ``attend`` for the words in ``kind``."""
    from hi3d_amd import attention

    g = torch.Generator().manual_seed(seed)
    kw = {}
    if "cap" in kind:
        kw["cap"] = 3.0
    if "slopes" in kind:
        kw["slopes"] = attention.head_slopes(heads)
    if "bias" in kind:
        kw["bias"] = torch.randn((count, heads), generator=g).to(dtype).cuda()
        kw["buckets"] = attention.relative_buckets(count, far, causal=causal)
    if "prefix" in kind:
        kw["prefix"] = torch.randint(0, longest + 1, (segments,), generator=g, dtype=torch.int32).cuda()
    return kw


def on_host(kw):
    """The same for the oracle (``prefix`` apart)."""
    return {"cap": kw.get("cap"), "slopes": host(kw.get("slopes")), "bias": host(kw.get("bias")),
            "buckets": None if kw.get("buckets") is None else kw["buckets"].cpu().numpy()}


def within(got, want, room, what):
    got = host(got)
    assert got.shape == want.shape, (got.shape, want.shape)
    assert np.isfinite(got).all(), f"{what} is not finite"
    off = np.abs(got - want)
    assert (off <= room).all(), f"{what}: {np.max(off / np.maximum(room, 1e-300))} of the room"


def check_rows(out, lse, f, dtype, what="out", for_grad=False):
    """One head's output ``[lq, d]`` and lse against ``oracle.attention_terms.head``'s ``f``.

    ``for_grad``: for gradients rows may be divided by the sum of the rounded probabilities, w_j = p_j (1 +
    t_j) with |t_j| <= u: sum_j w_j v_j / sum_j w_j is off from out by sum_j p_j t_j (v_j - out) / (1 +
    sum_j p_j t_j), at most u (sum_j p_j |v_j| + |out|) to first order: u |out| more than for the
    quotient with the sum of the p_j."""
    u, tiny = U[dtype], TINY[dtype]
    rounded = u * np.abs(f["out"]) * (2 if for_grad else 1)
    within(out, f["out"], f["out_off"] * 1.01 + u * f["size"] + tiny * f["vsum"] + rounded + 2 * tiny, what)
    if lse is not None:
        got, none = host(lse), np.isneginf(f["lse"])
        assert np.array_equal(np.isneginf(got), none)
        got, want = np.where(none, 0, got), np.where(none, 0, f["lse"])
        room = 1.01 * f["row"] + 4 * E * np.abs(want) + 8 * E
        assert (np.abs(got - want) <= room).all(), np.max(np.abs(got - want) / room)


def check(q, k, v, lengths_q, lengths_k=None, *, dout=None, dlse=None, mask=None, causal=False, scale=None, **kw):
    """Runs ``attend`` over packed segments (with ``dout`` its gradients too) and checks all of it."""
    from hi3d_amd import attention

    lengths_k = lengths_q if lengths_k is None else lengths_k
    one = len(lengths_q) == 1 and kw.get("prefix") is None and lengths_q[0] == len(q) and lengths_k[0] == len(k)
    cu = () if one else (attention.offsets(lengths_q), attention.offsets(lengths_k))
    leaves = [x.detach().requires_grad_(dout is not None) for x in (q, k, v)]
    call = dict(kw)
    if dout is not None and "bias" in kw:
        call["bias"] = kw["bias"].detach().requires_grad_(True)
        leaves.append(call["bias"])
    out, lse = attention.attend(*leaves[:3], *cu, causal=causal, key_mask=mask, scale=scale, return_lse=True, **call)
    grads = [None] * 4
    if dout is not None:
        outs, gs = ((out, lse), (dout, dlse)) if dlse is not None else ((out,), (dout,))
        grads = list(torch.autograd.grad(outs, leaves, gs)) + [None] * (4 - len(leaves))
    check_all(q, k, v, lengths_q, lengths_k, out, lse, grads, dout=dout, dlse=dlse, mask=mask, causal=causal, scale=scale, **kw)
    return out, lse, grads


def check_all(q, k, v, lengths_q, lengths_k, out, lse, grads, *, dout=None, dlse=None, mask=None, causal=False, scale=None, **kw):
    dtype, d, hq, hk = q.dtype, q.shape[-1], q.shape[-2], k.shape[-2]
    scale = d ** -0.5 if scale is None else scale
    ends_q, ends_k, prefix = ends(lengths_q), ends(lengths_k), host(kw.get("prefix"))
    qh, kh, vh, mh, dh, zh = host(q), host(k), host(v), host(mask), host(dout), host(dlse)
    on = on_host(kw)
    want = {n: np.zeros(x.shape) for n, x in (("dq", qh), ("dk", kh), ("dv", vh), ("dq_off", qh), ("dk_off", kh), ("dv_off", vh))}
    if dout is not None and on["bias"] is not None:
        want["dbias"], want["dbias_off"] = np.zeros(on["bias"].shape), np.zeros(on["bias"].shape)
    u, tiny, floor = U[dtype], TINY[dtype], 0.0
    if dout is not None and dtype == torch.float16:
        most = np.abs(dh).sum(-1).max(initial=0)
        if zh is not None:
            most = max(most, np.abs(zh).max(initial=0))
        floor = 2.0 ** -35 + 2.0 ** -28 * most
    for s, (a, b, c, e) in enumerate(zip(ends_q[:-1], ends_q[1:], ends_k[:-1], ends_k[1:])):
        if a == b:
            continue
        for h in range(hq):
            g = h // (hq // hk)
            pre = 0 if prefix is None else int(min(max(prefix[s], 0), e - c))
            f = oterms.head(qh[a:b, h], kh[c:e, g], vh[c:e, g], h, scale, causal, None if mh is None else mh[c:e] > 0, pre, **on)
            check_rows(out[a:b, h], None if lse is None else lse[a:b, h], f, dtype, f"out of segment {s} head {h}",
                       dout is not None)
            if dout is None or c == e:
                continue
            r = oterms.head_grad(f, qh[a:b, h], dh[a:b, h], scale, u + 4 * E, tiny, floor, None if zh is None else zh[a:b, h])
            for n in ("dq", "dq_off"):
                want[n][a:b, h] = r[n]
            for n in ("dk", "dv", "dk_off", "dv_off"):
                want[n][c:e, g] += r[n]
            if "dbias" in want:
                far = (len(on["buckets"]) - 1) // 2
                at = np.clip(on["buckets"], 0, len(on["bias"]) - 1)[np.clip(oterms.positions(b - a, e - c), -far, far) + far]
                for n, x in (("dbias", r["ds"]), ("dbias_off", r["ds_off"] + floor * f["seen"])):
                    want[n][:, h] += np.bincount(at.ravel(), x.ravel(), len(on["bias"]))
    for got, n in zip(grads, ("dq", "dk", "dv", "dbias")):
        if got is None:
            continue
        ug = U[got.dtype]
        # sums by relative position over n pairs in fp32: n / 64 e of their magnitudes (64 lanes and tiles apart)
        within(got, want[n], 1.01 * want[n + "_off"] + ug * np.abs(want[n]) + 2 * TINY[got.dtype], n)
