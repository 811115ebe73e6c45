"""Attention and its gradients in float64 from the definition, segment by segment, with
the magnitudes that bound a kernel's rounding errors (the torso's self attention,
src/sparc3d/nn/sparse/attention/full_attn.py:35-77)."""

from __future__ import annotations

import numpy as np


def spans(cu) -> list[tuple[int, int]]:
    return [(int(a), int(b)) for a, b in zip(cu[:-1], cu[1:])]


def _visible(lq: int, lk: int, causal: bool, mask) -> np.ndarray:
    seen = np.ones((lq, lk), bool)
    if causal:
        seen &= np.arange(lk)[None, :] <= np.arange(lq)[:, None] + (lk - lq)
    if mask is not None:
        seen &= np.asarray(mask, bool)[None, :]
    return seen


def _head(q, k, v, scale, seen):
    """``p [lq, lk]``, ``out``, ``lse`` of one head; hidden keys are left out, not multiplied."""
    k, v = np.where(seen.any(0)[:, None], k, 0.0), np.where(seen.any(0)[:, None], v, 0.0)
    s = np.where(seen, scale * (q @ k.T), -np.inf)
    top = np.where(seen.any(1), s.max(1, initial=-np.inf), 0.0)
    e = np.exp(s - top[:, None])
    total = e.sum(1)
    p = e / np.where(total > 0, total, 1.0)[:, None]
    with np.errstate(divide="ignore"):
        return k, v, p, p @ v, top + np.log(total)


def forward(q, k, v, segments_q, segments_k, scale=None, causal=False, mask=None) -> dict:
    """``q [Nq, hq, d]``, ``k`` / ``v [Nk, hk, d]``; ``segments``: (begin, end) rows. Returns
    ``out``, ``lse``, ``size`` = ``sum_j p_j |v_j|``, ``vsum`` = ``sum_j |v_j|`` over visible
    keys and ``reach`` = ``scale * max_j sum_d |q_d k_jd|`` (what an fp32 score can be off by,
    in units of its rounding)."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    hq, hk, d = q.shape[1], k.shape[1], q.shape[2]
    scale = d ** -0.5 if scale is None else scale
    r = {"out": np.zeros(q.shape), "lse": np.full(q.shape[:2], -np.inf), "size": np.zeros(q.shape),
         "vsum": np.zeros(q.shape), "reach": np.zeros(q.shape[:2])}
    for (q0, q1), (k0, k1) in zip(segments_q, segments_k):
        if q1 == q0 or k1 == k0:
            continue
        seen = _visible(q1 - q0, k1 - k0, causal, None if mask is None else mask[k0:k1])
        for h in range(hq):
            g = h // (hq // hk)
            kk, vv, p, out, lse = _head(q[q0:q1, h], k[k0:k1, g], v[k0:k1, g], scale, seen)
            r["out"][q0:q1, h], r["lse"][q0:q1, h] = out, lse
            r["size"][q0:q1, h], r["vsum"][q0:q1, h] = p @ np.abs(vv), seen @ np.abs(vv)
            r["reach"][q0:q1, h] = scale * (np.abs(q[q0:q1, h]) @ np.abs(kk).T).max(1)
    return r


def backward(q, k, v, dout, segments_q, segments_k, scale=None, causal=False, mask=None, delta_error=None,
             p_error=0.0, u=0.0, floor=0.0, dlse=None) -> dict:
    """``dq``, ``dk``, ``dv`` and bounds ``dq_off``, ``dk_off``, ``dv_off`` of their errors when
    probabilities and score gradients are rounded to a relative ``u`` (absolute ``floor``)
    before their products, a row's ``sum(dout * out)`` is off by ``delta_error [Nq, hq]`` and
    a probability by a relative ``p_error [Nq, hq]``. ``dlse [Nq, hq]``: the gradient of ``lse``."""
    q, k, v, dout = (np.asarray(x, np.float64) for x in (q, k, v, dout))
    hq, hk, d = q.shape[1], k.shape[1], q.shape[2]
    scale = d ** -0.5 if scale is None else scale
    r = {n: np.zeros(x.shape) for n, x in (("dq", q), ("dk", k), ("dv", v), ("dq_off", q), ("dk_off", k), ("dv_off", v))}
    for (q0, q1), (k0, k1) in zip(segments_q, segments_k):
        if q1 == q0 or k1 == k0:
            continue
        seen = _visible(q1 - q0, k1 - k0, causal, None if mask is None else mask[k0:k1])
        for h in range(hq):
            g = h // (hq // hk)
            qq, do = q[q0:q1, h], dout[q0:q1, h]
            kk, vv, p, out, _ = _head(qq, k[k0:k1, g], v[k0:k1, g], scale, seen)
            dp = do @ vv.T
            inner = dp - (do * out).sum(1)[:, None]
            if dlse is not None:
                inner = inner + np.asarray(dlse, np.float64)[q0:q1, h][:, None]
            inner = np.where(seen, inner, 0.0)
            ds = p * inner
            r["dq"][q0:q1, h] = scale * ds @ kk
            r["dk"][k0:k1, g] += scale * ds.T @ qq
            r["dv"][k0:k1, g] += p.T @ do
            if delta_error is None:
                continue
            pe = np.broadcast_to(np.asarray(p_error), q.shape[:2])[q0:q1, h][:, None]
            p_off = np.where(seen, p * (u + pe) + floor, 0.0)
            dp_off = d * 2.0 ** -24 * (np.abs(do) @ np.abs(vv).T)
            ds_off = np.where(seen, np.abs(ds) * (u + pe) + floor + p * (delta_error[q0:q1, h][:, None] + dp_off), 0.0)
            r["dq_off"][q0:q1, h] = scale * ds_off @ np.abs(kk)
            r["dk_off"][k0:k1, g] += scale * ds_off.T @ np.abs(qq)
            r["dv_off"][k0:k1, g] += p_off.T @ np.abs(do)
    return r
