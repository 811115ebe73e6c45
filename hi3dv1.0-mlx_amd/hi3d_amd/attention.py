"""Attention over packed segments of tokens: ``softmax(scale * q k^T) v``.

Tokens of all sequences (objects of a batch, windows of a serialized level) follow one
another in ``[N, heads, dim]`` with int32 offsets of where each begins, or lie in equal room
``[B, L, heads, dim]``. fp16 or bf16, head sizes that are multiples of 8 up to 128, query
heads in groups over fewer key heads. fp32 scores, sums and accumulation.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib


class _Desc(ctypes.Structure):
    """``hi3d_attention_desc``."""

    _fields_ = [
        *[(n, ctypes.c_void_p) for n in ("q", "k", "v", "cu_q", "cu_k", "lens_k", "key_mask")],
        ("strides", ctypes.c_int64 * 9), ("total_q", ctypes.c_int64), ("total_k", ctypes.c_int64),
        *[(n, ctypes.c_int32) for n in ("batch", "len_q", "len_k", "heads_q", "heads_k", "dim", "dtype", "causal")],
        ("scale", ctypes.c_float),
    ]


def offsets(lengths, device: torch.device | str = "cuda") -> torch.Tensor:
    """int32 offsets ``[len(lengths) + 1]`` of segments of the given lengths."""
    at = [0]
    for n in lengths:
        if int(n) < 0:
            raise ValueError(f"a segment of {n} tokens")
        at.append(at[-1] + int(n))
    if at[-1] >= 1 << 31:
        raise ValueError("offsets must fit in 31 bits")
    return torch.tensor(at, dtype=torch.int32).to(device)


def _heads(x: torch.Tensor) -> torch.Tensor:
    """``x`` itself where the kernels can read it (adjacent values, 16-byte aligned heads and
    rows, non-negative strides below 2^23), else a copy."""
    inner = x.dim() - 2
    ok = (x.shape[-1] == 1 or x.stride(-1) == 1) and x.data_ptr() % 16 == 0
    ok = ok and all(s % 8 == 0 for s in x.stride()[:-1]) and x.stride(inner - 1) < 1 << 23
    if ok:
        return x
    x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


def _offsets_of(cu: torch.Tensor | None, what: str) -> torch.Tensor | None:
    if cu is None:
        return None
    if cu.dim() != 1 or cu.dtype not in (torch.int32, torch.int64) or cu.numel() < 1:
        raise ValueError(f"{what} must be int32 offsets [segments + 1]")
    return cu.to(torch.int32).contiguous()


class _Problem:
    """One checked attention problem: the descriptor and the tensors it points into."""

    def __init__(self, q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask):
        for name, x in (("q", q), ("k", k), ("v", v)):
            if x.dim() != q.dim() or x.dim() not in (3, 4):
                raise ValueError(f"{name} must be [tokens, heads, dim], or [batch, length, heads, dim] like the others")
            if x.dtype != q.dtype:
                raise ValueError(f"q, k and v of different types: {q.dtype} and {x.dtype}")
        if q.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"attention takes fp16 or bf16 (got {q.dtype})")
        if k.shape != v.shape:
            raise ValueError(f"keys {list(k.shape)} and values {list(v.shape)} differ")
        dim, hq, hk = int(q.shape[-1]), int(q.shape[-2]), int(k.shape[-2])
        if k.shape[-1] != dim:
            raise ValueError(f"heads of {dim} and {k.shape[-1]} values")
        if dim % 8 or not 8 <= dim <= 128:
            raise ValueError(f"head size must be a multiple of 8 up to 128 (got {dim})")
        if hk < 1 or hq < 1 or hq % hk:
            raise ValueError(f"{hq} query heads are no multiple of {hk} key heads")
        scale = dim ** -0.5 if scale is None else float(scale)
        if not (scale > 0 and math.isfinite(scale)):
            raise ValueError("scale must be positive and finite")
        cu_q, cu_k = _offsets_of(cu_q, "cu_q"), _offsets_of(cu_k, "cu_k")
        if q.dim() == 4:
            if cu_q is not None or cu_k is not None:
                raise ValueError("offsets belong to packed tokens [tokens, heads, dim]")
            if q.shape[0] != k.shape[0]:
                raise ValueError(f"{q.shape[0]} and {k.shape[0]} batch elements")
            batch, len_q, len_k = int(q.shape[0]), int(q.shape[1]), int(k.shape[1])
        else:
            if cu_k is None and cu_q is not None:
                if q.shape[0] != k.shape[0]:
                    raise ValueError("keys of other segments than the queries' need offsets of their own")
                cu_k = cu_q
            if (cu_q is None) != (cu_k is None) or (cu_q is not None and cu_q.numel() != cu_k.numel()):
                raise ValueError("queries and keys need offsets of the same segments")
            batch, len_q, len_k = 1, int(q.shape[0]), int(k.shape[0])
            if cu_q is not None:
                batch, len_q, len_k = cu_q.numel() - 1, 0, 0
                if batch == 0 and (q.shape[0] or k.shape[0]):
                    raise ValueError("tokens without a segment")
        if lens_k is not None:
            if q.dim() != 4 or lens_k.shape != (batch,) or lens_k.dtype not in (torch.int32, torch.int64):
                raise ValueError("lens_k must be int32 [batch], for tokens [batch, length, heads, dim]")
            lens_k = lens_k.to(torch.int32).contiguous()
        if key_mask is not None:
            if key_mask.dtype not in (torch.bool, torch.uint8) or key_mask.shape != k.shape[:-2]:
                raise ValueError(f"key_mask must be bool {list(k.shape[:-2])}")
            key_mask = key_mask.contiguous()
        self.device = _lib.require_gpu(q, k, v, cu_q, cu_k, lens_k, key_mask)
        q, k, v = _heads(q), _heads(k), _heads(v)
        self.keep = (q, k, v, cu_q, cu_k, lens_k, key_mask)
        d = self.desc = _Desc()
        d.q, d.k, d.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
        d.cu_q, d.cu_k, d.lens_k, d.key_mask = (_lib.ptr(t) for t in (cu_q, cu_k, lens_k, key_mask))
        strides = []
        for x in (q, k, v):
            strides += [0, *x.stride()[:-1]] if x.dim() == 3 else x.stride()[:-1]
        d.strides[:] = strides
        d.total_q, d.total_k = q.numel() // (hq * dim), k.numel() // (hk * dim)
        d.batch, d.len_q, d.len_k, d.heads_q, d.heads_k, d.dim = batch, len_q, len_k, hq, hk, dim
        d.dtype, d.causal, d.scale = _lib.DTYPES[q.dtype], int(bool(causal)), scale

    def forward(self, want_lse: bool) -> tuple[torch.Tensor, torch.Tensor | None]:
        q = self.keep[0]
        out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=self.device) if want_lse else None
        need = _lib.query("hi3d_attention_workspace", ctypes.byref(self.desc))
        work = _lib.workspace(need, self.device) if need else None
        _lib.call("hi3d_attention_forward", ctypes.byref(self.desc), _lib.ptr(out), _lib.ptr(lse), _lib.ptr(work), need,
                  _lib.stream(self.device))
        return out, lse


    def backward(self, out, lse, dout, dlse, want_q: bool, want_kv: bool):
        q, k = self.keep[:2]
        self.dense = [x if x is None else _dense(x) for x in (out, lse, dout, dlse)]
        out, lse, dout, dlse = self.dense
        dq = torch.empty(q.shape, dtype=q.dtype, device=self.device) if want_q else None
        dk = torch.empty(k.shape, dtype=k.dtype, device=self.device) if want_kv else None
        dv = torch.empty(k.shape, dtype=k.dtype, device=self.device) if want_kv else None
        need = _lib.query("hi3d_attention_backward_workspace", ctypes.byref(self.desc))
        work = _lib.workspace(need, self.device) if need else None
        _lib.call("hi3d_attention_backward", ctypes.byref(self.desc), out.data_ptr(), lse.data_ptr(), dout.data_ptr(),
                  _lib.ptr(dlse), _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv), _lib.ptr(work), need, _lib.stream(self.device))
        return dq, dk, dv


def _dense(x: torch.Tensor) -> torch.Tensor:
    x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask):
        p = _Problem(q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask)
        out, lse = p.forward(True)
        ctx.save_for_backward(q, k, v, cu_q, cu_k, lens_k, key_mask, out, lse)
        ctx.how = (scale, causal)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dlse):
        q, k, v, cu_q, cu_k, lens_k, key_mask, out, lse = ctx.saved_tensors
        want_q, want_kv = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        if (dout is None and dlse is None) or not (want_q or want_kv):
            return (None,) * 9
        dout = torch.zeros_like(out) if dout is None else dout
        p = _Problem(q, k, v, cu_q, cu_k, lens_k, *ctx.how, key_mask)
        with torch.cuda.device(p.device):
            dq, dk, dv = p.backward(out, lse, dout, dlse, want_q, want_kv)
        return dq, dk, dv, None, None, None, None, None, None


def attend(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_q: torch.Tensor | None = None,
    cu_k: torch.Tensor | None = None,
    *,
    lens_k: torch.Tensor | None = None,
    scale: float | None = None,
    causal: bool = False,
    key_mask: torch.Tensor | None = None,
    return_lse: bool = False,
):
    """``softmax(scale * q k^T) v`` within each segment, ``scale`` = ``dim ** -0.5`` by default.

    ``q [Nq, hq, dim]``, ``k`` and ``v [Nk, hk, dim]`` with offsets ``cu_q`` / ``cu_k`` (int32,
    ascending from 0 to ``Nq`` / ``Nk``; ``cu_k`` = ``cu_q`` by default; one segment without
    offsets), or ``[B, L, heads, dim]``, where ``lens_k [B]`` says how many keys of each are in
    use (a cache). Query head ``h`` reads key head ``h // (hq // hk)``. ``causal``: query ``i``
    of ``lq`` sees the keys ``j <= i + lk - lq`` (a later key whose value is not finite can still
    reach it: such keys belong in ``key_mask``). ``key_mask`` (bool, one per key): False keys
    are not seen, whatever they hold. A row that sees no key gives zeros. Views with other
    strides are read in place where their rows are 16-byte aligned.

    Returns ``[..., hq, dim]`` (and with ``return_lse`` the float32 ``log(sum(exp(scores)))``
    per row and head, -inf for a row that sees no key). Differentiable once in ``q``, ``k`` and
    ``v``, through both outputs; :func:`attend_grad` is the same without autograd."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _Attend.apply(q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask)
        return (out, lse) if return_lse else out
    p = _Problem(q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask)
    with torch.cuda.device(p.device):
        out, lse = p.forward(return_lse)
    return (out, lse) if return_lse else out


def attend_grad(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    out: torch.Tensor,
    lse: torch.Tensor,
    dout: torch.Tensor,
    cu_q: torch.Tensor | None = None,
    cu_k: torch.Tensor | None = None,
    *,
    dlse: torch.Tensor | None = None,
    lens_k: torch.Tensor | None = None,
    scale: float | None = None,
    causal: bool = False,
    key_mask: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``dq``, ``dk`` and ``dv`` of :func:`attend` from its arguments, its ``out`` and ``lse``, the
    gradient ``dout`` of ``out`` and optionally ``dlse`` of ``lse``.

    Sums run in a fixed order: the same bits every time. fp32 sums; probabilities and score
    gradients are rounded once to the inputs' type for their products (in fp16 after a scaling
    by powers of two, so that small gradients of long rows keep their digits). Launches only:
    this is the form to capture into a graph, with no autograd node of another stream in it."""
    p = _Problem(q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask)
    for name, x, shape, dtype in (("out", out, q.shape, q.dtype), ("dout", dout, q.shape, q.dtype),
                                  ("lse", lse, q.shape[:-1], torch.float32), ("dlse", dlse, q.shape[:-1], torch.float32)):
        if x is not None and (x.shape != shape or x.dtype != dtype):
            raise ValueError(f"{name} must be {list(shape)} of {dtype} (got {list(x.shape)} of {x.dtype})")
    _lib.require_gpu(q, out, lse, dout, dlse)
    with torch.cuda.device(p.device), torch.no_grad():
        return p.backward(out, lse, dout, dlse, True, True)
