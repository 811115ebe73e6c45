"""Attention whose scores carry terms, and its gradients, in float64 from the definition, with
bounds of what a kernel's roundings can move (``e`` = 2^-24):

* a score: (d + 4) e scale sum |q k| for its product, 10 e cap for the cap (an exponential and a
  reciprocal of 1 ulp each, a sum and a multiply-add; its derivative is at most 1), 8 e (slope
  (|r| + 64) + |bias|) for multiply-adds that take a tile's distances apart, and 4 e (|s| +
  |largest s|) in the exponent;
* a row's sum and lse: the same, weighed by the probabilities, and (16 + keys) e.
"""

from __future__ import annotations

import numpy as np

E = 2.0 ** -24
HIDE_BELOW = -1e5
"""A bias below hides its keys."""
LOST_BELOW = -(2.0 ** 22) * np.log(2.0)
"""A row whose largest score is below sees no key."""


def positions(lq: int, lk: int) -> np.ndarray:
    """Key ``j`` relative to query ``i``, the last query at the last key."""
    return np.arange(lk)[None, :] - (np.arange(lq)[:, None] + lk - lq)


def _scores(q, k, head, scale, r, seen, cap, slopes, bias, buckets):
    """Scores, the cap's derivative, and the bound of a score's error."""
    d = q.shape[1]
    x = scale * (q @ k.T)
    off = (d + 4) * E * scale * (np.abs(q) @ np.abs(k).T)
    bend = np.ones_like(x)
    if cap:
        t = np.tanh(x / cap)
        x, bend, off = cap * t, 1 - t * t, off + 10 * E * cap
    if slopes is not None:
        x, off = x - slopes[head] * np.abs(r), off + 8 * E * slopes[head] * (np.abs(r) + 64)
    if bias is not None:
        far = (len(buckets) - 1) // 2
        b = bias[np.clip(buckets, 0, len(bias) - 1)[np.clip(r, -far, far) + far], head]
        seen = seen & ~(b < HIDE_BELOW)
        b = np.where(seen, b, 0.0)
        x, off = x + b, off + 8 * E * np.abs(b)
    x = np.where(seen, x, -np.inf)
    seen = seen & (x.max(1, initial=-np.inf) >= LOST_BELOW)[:, None]
    x = np.where(seen, x, -np.inf)
    return x, bend, np.where(seen, off, 0.0), seen


def _softmax(x, off, seen):
    some = seen.any(1)
    top = np.where(some, x.max(1, initial=-np.inf), 0.0)
    w = np.exp(x - top[:, None])
    total = w.sum(1)
    p = w / np.where(total > 0, total, 1.0)[:, None]
    with np.errstate(divide="ignore"):
        lse = top + np.log(total)
    size = np.where(seen, np.abs(np.where(seen, x, 0.0)), 0.0)
    off = np.where(seen, off + 4 * E * (size + np.abs(top)[:, None]), 0.0)
    row = (p * off).sum(1) + (16 + x.shape[1]) * E
    return p, lse, off, row


def seen_keys(lq: int, lk: int, causal: bool, mask, prefix: int) -> np.ndarray:
    seen = np.ones((lq, lk), bool)
    if causal:
        seen &= (positions(lq, lk) <= 0) | (np.arange(lk) < prefix)[None, :]
    if mask is not None:
        seen &= np.asarray(mask, bool)[None, :]
    return seen


def head(q, k, v, which, scale=None, causal=False, mask=None, prefix=0, r=None, seen=None, cap=None, slopes=None, bias=None,
         buckets=None) -> dict:
    """One query head ``which`` of one segment: ``q [lq, d]``, ``k`` and ``v [lk, d]``. ``out``, ``lse``,
    ``p``, ``bend`` (the cap's derivative), ``size`` = p |v|, ``vsum`` = sums of the seen |v|, and bounds:
    ``off`` of the scores, ``row`` of a row's sum, ``out_off`` of the output before any rounding to 16
    bits. ``r`` and ``seen`` stand in for a segment's own."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    lq, lk = len(q), len(k)
    scale = q.shape[1] ** -0.5 if scale is None else scale
    r = positions(lq, lk) if r is None else r
    seen = seen_keys(lq, lk, causal, mask, prefix) if seen is None else seen
    any_row = seen.any(0)[:, None]
    k, v = np.where(any_row, k, 0.0), np.where(any_row, v, 0.0)
    x, bend, off, seen = _scores(q, k, which, scale, r, seen, cap, slopes, bias, buckets)
    p, lse, off, row = _softmax(x, off, seen)
    size = p @ np.abs(v)
    return {"out": p @ v, "lse": lse, "p": p, "bend": bend, "size": size, "vsum": seen @ np.abs(v), "off": off, "row": row,
            "out_off": (p * off) @ np.abs(v) + row[:, None] * size, "seen": seen, "k": k, "v": v}


def head_grad(f: dict, q, dout, scale, u: float, tiny: float, floor: float, dlse=None) -> dict:
    """Gradients of one head from :func:`head`'s ``f``: ``dq``, ``dk``, ``dv``, ``ds`` (of the scores, for
    the bias) and their bounds ``.._off`` when p and ds are rounded to a relative ``u`` (absolute
    ``floor``) for their products and the output, of which D is formed, to ``u`` (``tiny``)."""
    q, do = np.asarray(q, np.float64), np.asarray(dout, np.float64)
    k, v, p = f["k"], f["v"], f["p"]
    d = q.shape[1]
    inner = do @ v.T - (do * f["out"]).sum(1)[:, None]
    if dlse is not None:
        inner = inner + np.asarray(dlse, np.float64)[:, None]
    ds = p * np.where(f["seen"], inner, 0.0)
    out_off = f["out_off"] + u * f["size"] + tiny * f["vsum"] + u * np.abs(f["out"]) + 2 * tiny
    delta = (np.abs(do) * out_off).sum(1) + (d + 1) * E * (np.abs(do) * np.abs(f["out"])).sum(1)
    lse = np.abs(np.where(np.isneginf(f["lse"]), 0.0, f["lse"]))
    pe = f["off"] + f["row"][:, None] + 14 * E * (1 + lse)[:, None]
    sums = (len(q) + len(k)) / 16 * E
    ds_off = np.abs(ds) * (pe + sums) + p * (delta[:, None] + d * E * (np.abs(do) @ np.abs(v).T))
    dx = ds * f["bend"]
    dx_off = np.where(f["seen"], ds_off * f["bend"] + 12 * E * np.abs(ds) + np.abs(dx) * u + floor, 0.0)
    p_off = np.where(f["seen"], p * (u + pe + sums) + floor, 0.0)
    return {"dq": scale * dx @ k, "dk": scale * dx.T @ q, "dv": p.T @ do, "ds": ds, "ds_off": ds_off,
            "dq_off": scale * dx_off @ np.abs(k), "dk_off": scale * dx_off.T @ np.abs(q), "dv_off": p_off.T @ np.abs(do)}
