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


def _heads(x: torch.Tensor) -> tuple[torch.Tensor, tuple[int, ...]]:
    """``x`` itself where the kernels can read it (adjacent values, 16-byte aligned heads and
    rows, non-negative strides below 2^23), else a copy; and its strides."""
    strides = x.stride()
    if (strides[-1] == 1 or x.shape[-1] == 1) and strides[-3] < 1 << 23 and not x.data_ptr() % 16:
        bits = strides[-2] | strides[-3]
        if not (bits | strides[0]) % 8:
            return x, strides
    if 1 in x.shape[:-1]:  # the stride of a dimension of one says nothing, and contiguous() leaves it
        if any(s and n == 1 for s, n in zip(strides, x.shape)):
            return _heads(x.as_strided(x.shape, [0 if n == 1 else s for s, n in zip(strides, x.shape)]))
    x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone()
    return x, [0 if n == 1 else s for s, n in zip(x.stride(), x.shape)]


def _offsets_of(cu: torch.Tensor, what: str) -> torch.Tensor:
    if cu.dim() != 1 or cu.dtype not in (torch.int32, torch.int64) or cu.numel() < 1:
        raise ValueError(f"{what} must be int32 offsets [segments + 1]")
    return cu if cu.dtype == torch.int32 and cu.is_contiguous() else cu.to(torch.int32).contiguous()


class _Problem:
    """One checked attention problem: the descriptor and the tensors it points into."""

    def __init__(self, q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask):
        shape, key_shape, dtype = q.shape, k.shape, q.dtype
        rank = len(shape)
        for name, x in (("q", q), ("k", k), ("v", v)):
            if x.dim() != rank or rank not in (3, 4):
                raise ValueError(f"{name} must be [tokens, heads, dim], or [batch, length, heads, dim] like the others")
            if x.dtype != dtype:
                raise ValueError(f"q, k and v of different types: {dtype} and {x.dtype}")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"attention takes fp16 or bf16 (got {dtype})")
        if key_shape != v.shape:
            raise ValueError(f"keys {list(key_shape)} and values {list(v.shape)} differ")
        dim, hq, hk = shape[-1], shape[-2], key_shape[-2]
        if key_shape[-1] != dim:
            raise ValueError(f"heads of {dim} and {key_shape[-1]} values")
        if dim % 8 or not 8 <= dim <= 128:
            raise ValueError(f"head size must be a multiple of 8 up to 128 (got {dim})")
        if hk < 1 or hq < 1 or hq % hk:
            raise ValueError(f"{hq} query heads are no multiple of {hk} key heads")
        scale = dim ** -0.5 if scale is None else float(scale)
        if not (scale > 0 and math.isfinite(scale)):
            raise ValueError("scale must be positive and finite")
        if cu_q is not None:
            cu_q = _offsets_of(cu_q, "cu_q")
        if cu_k is not None:
            cu_k = _offsets_of(cu_k, "cu_k")
        if rank == 4:
            if cu_q is not None or cu_k is not None:
                raise ValueError("offsets belong to packed tokens [tokens, heads, dim]")
            batch, len_q, len_k = shape[0], shape[1], key_shape[1]
            if key_shape[0] != batch:
                raise ValueError(f"{batch} and {key_shape[0]} batch elements")
            total_q, total_k = batch * len_q, batch * len_k
        else:
            total_q, total_k = shape[0], key_shape[0]
            if cu_k is None and cu_q is not None:
                if total_q != total_k:
                    raise ValueError("keys of other segments than the queries' need offsets of their own")
                cu_k = cu_q
            if (cu_q is None) != (cu_k is None) or (cu_q is not None and cu_q.numel() != cu_k.numel()):
                raise ValueError("queries and keys need offsets of the same segments")
            batch, len_q, len_k = 1, total_q, total_k
            if cu_q is not None:
                batch, len_q, len_k = cu_q.numel() - 1, 0, 0
                if batch == 0 and (total_q or total_k):
                    raise ValueError("tokens without a segment")
        if lens_k is not None:
            if rank != 4 or lens_k.shape != (batch,) or lens_k.dtype not in (torch.int32, torch.int64):
                raise ValueError("lens_k must be int32 [batch], for tokens [batch, length, heads, dim]")
            lens_k = lens_k.to(torch.int32).contiguous()
        if key_mask is not None:
            if key_mask.dtype not in (torch.bool, torch.uint8) or key_mask.shape != key_shape[:-2]:
                raise ValueError(f"key_mask must be bool {list(key_shape[:-2])}")
            key_mask = key_mask.contiguous()
        self.device = _lib.require_gpu(q, k, v, cu_q, cu_k, lens_k, key_mask)
        self.set((q, k, v, cu_q, cu_k, lens_k, key_mask),
                 (total_q, total_k, batch, len_q, len_k, hq, hk, dim, _lib.DTYPES[dtype], 1 if causal else 0, scale))

    @classmethod
    def again(cls, tensors, sizes) -> _Problem:
        """A problem that was checked before, of its ``tensors`` (or copies of them) and ``sizes``."""
        p = cls.__new__(cls)
        p.device = tensors[0].device
        p.set(tensors, sizes)
        return p

    def set(self, tensors, sizes) -> None:
        (q, q_s), (k, k_s), (v, v_s) = _heads(tensors[0]), _heads(tensors[1]), _heads(tensors[2])
        self.tensors, self.sizes = (q, k, v, *tensors[3:]), sizes
        strides = (0, *q_s[:2], 0, *k_s[:2], 0, *v_s[:2]) if len(q_s) == 3 else (*q_s[:3], *k_s[:3], *v_s[:3])
        self.desc = _Desc(*[x if x is None else x.data_ptr() for x in self.tensors], strides, *sizes)
        self.ref = ctypes.byref(self.desc)

    def forward(self, want_lse: bool) -> tuple[torch.Tensor, torch.Tensor | None]:
        q, ref = self.tensors[0], self.ref
        out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=self.device) if want_lse else None
        need = _lib.query("hi3d_attention_workspace", ref)
        work = _lib.workspace(need, self.device) if need else None
        _lib.call("hi3d_attention_forward", ref, out.data_ptr(), _lib.ptr(lse), _lib.ptr(work), need,
                  _lib.stream(self.device))
        return out, lse

    def backward(self, out, lse, dout, dlse, want_q: bool, want_kv: bool):
        q, k = self.tensors[:2]
        if (q.shape[-2] // k.shape[-2] - 1) * q.stride(-2) >= 1 << 29:  # a tile's queries are addressed with 32 bits
            self.set((q.contiguous(), *self.tensors[1:]), self.sizes)
        ref = self.ref
        out, lse, dout = _dense(out), _dense(lse), _dense(dout)
        dlse = dlse if dlse is None else _dense(dlse)
        dq = torch.empty(q.shape, dtype=q.dtype, device=self.device) if want_q else None
        dk = torch.empty(k.shape, dtype=k.dtype, device=self.device) if want_kv else None
        dv = torch.empty(k.shape, dtype=k.dtype, device=self.device) if want_kv else None
        need = _lib.query("hi3d_attention_backward_workspace", ref)
        work = _lib.workspace(need, self.device) if need else None
        _lib.call("hi3d_attention_backward", ref, out.data_ptr(), lse.data_ptr(), dout.data_ptr(),
                  _lib.ptr(dlse), _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv), _lib.ptr(work), need, _lib.stream(self.device))
        return dq, dk, dv


def _dense(x: torch.Tensor) -> torch.Tensor:
    x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask):
        p = _Problem(q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask)
        with _lib.on(p.device):
            out, lse = p.forward(True)
        ctx.save_for_backward(*p.tensors, out, lse)
        ctx.sizes = p.sizes
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    def backward(ctx, dout, dlse):
        if torch.is_grad_enabled():
            raise RuntimeError("attention is differentiable once")
        want_q, want_kv = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        if (dout is None and dlse is None) or not (want_q or want_kv):
            return (None,) * 9
        *tensors, out, lse = ctx.saved_tensors
        dout = torch.zeros_like(out) if dout is None else dout
        p = _Problem.again(tensors, ctx.sizes)
        with _lib.on(p.device):
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
    ascending, within ``Nq`` / ``Nk``; ``cu_k`` = ``cu_q`` by default; one segment without
    offsets; rows before the first offset and from the last one on give zeros and take no
    part), or ``[B, L, heads, dim]``, where ``lens_k [B]`` says how many keys of each are in use
    (a cache). Query head ``h`` reads key head ``h // (hq // hk)``. ``causal``: query ``i``
    of ``lq`` sees the keys ``j <= i + lk - lq`` (a later key whose value is not finite can still
    reach it: such keys belong in ``key_mask``). ``key_mask`` (bool, one per key): False keys
    are not seen, whatever they hold. A row that sees no key gives zeros. Views with other
    strides are read in place where their rows are 16-byte aligned.

    Returns ``[..., hq, dim]`` (and with ``return_lse`` the float32 ``log(sum(exp(scores)))``
    per row and head, -inf for a row that sees no key). Differentiable once in ``q``, ``k`` and
    ``v`` (reverse mode), through both outputs; :func:`attend_grad` is the same without autograd
    (and says for which values fp16 gradients are formed)."""
    _lib.no_tangents("attention", q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _Attend.apply(q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask)
        return (out, lse) if return_lse else out
    p = _Problem(q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask)
    with _lib.on(p.device):
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
    by powers of two, so that small gradients of long rows keep their digits; with values of 8190
    and more that scaling can leave fp16's range, and the gradients of such a row are not finite
    then: take bf16 there). Launches only:
    this is the form to capture into a graph, with no autograd node of another stream in it."""
    _lib.no_tangents("attention", q, k, v, out, lse, dout, dlse)
    p = _Problem(q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask)
    for name, x, shape, dtype in (("out", out, q.shape, q.dtype), ("dout", dout, q.shape, q.dtype),
                                  ("lse", lse, q.shape[:-1], torch.float32), ("dlse", dlse, q.shape[:-1], torch.float32)):
        if x is not None and (x.shape != shape or x.dtype != dtype):
            raise ValueError(f"{name} must be {list(shape)} of {dtype} (got {list(x.shape)} of {x.dtype})")
    _lib.require_gpu(q, out, lse, dout, dlse)
    with _lib.on(p.device), torch.no_grad():
        return p.backward(out, lse, dout, dlse, True, True)
