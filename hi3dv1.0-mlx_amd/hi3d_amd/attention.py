"""Attention over packed segments of tokens: ``softmax(scale * q k^T) v``.

Tokens of all sequences (objects of a batch, windows of a serialized level) follow one
another in ``[N, heads, dim]`` with int32 offsets of where each begins, or lie in equal room
``[B, L, heads, dim]``. fp16 or bf16, head sizes that are multiples of 8 up to 128, query
heads in groups over fewer key heads. fp32 scores, sums and accumulation.

Scores may carry terms besides (:func:`attend`): a cap, a cost of distance, a learned bias by
relative position, a beginning that all queries of a causal segment see. :func:`attend_shared` is
for sequences that share their first keys.
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


class _TermsDesc(ctypes.Structure):
    """``hi3d_attention_terms``."""

    _fields_ = [
        *[(n, ctypes.c_void_p) for n in ("slopes", "bias", "bucket_map", "prefix")],
        *[(n, ctypes.c_int32) for n in ("bias_dtype", "buckets", "far")], ("cap", ctypes.c_float),
    ]


class _SharedDesc(ctypes.Structure):
    """``hi3d_attention_shared``."""

    _fields_ = [*[(n, ctypes.c_void_p) for n in ("k", "v", "key_mask")], ("strides", ctypes.c_int64 * 4),
                ("len", ctypes.c_int32)]


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


def head_slopes(heads: int, device: torch.device | str = "cuda") -> torch.Tensor:
    """float32 ``[heads]``: ``2 ** (-8 (h + 1) / heads)``, what a key of distance one costs in each head."""
    if heads < 1:
        raise ValueError(f"{heads} heads")
    return (2.0 ** (-8.0 * torch.arange(1, heads + 1, dtype=torch.float64) / heads)).float().to(device)


def relative_buckets(count: int, far: int, *, causal: bool = False, device: torch.device | str = "cuda") -> torch.Tensor:
    """int32 ``[2 far + 1]``: which of ``count`` buckets a relative position ``-far .. far`` (key minus
    query) belongs to. Each side has half of them (with ``causal`` keys before have all, and later ones
    count as distance 0); of a side's, the first half are distances of their own, and the others
    reach ``far`` with distances that grow by a constant factor."""
    side = count if causal else count // 2
    near = side // 2
    if side < 2 or not causal and count % 2:
        raise ValueError(f"an even number of at least 4 buckets, or 2 of one side (got {count})")
    if not near < far <= _FAR:
        raise ValueError(f"far must be above {near} and at most {_FAR} (got {far})")
    rest, place = side - near, list(range(near))
    for d in range(near, far + 1):  # the largest n with d >= near (far / near) ** (n / rest), in whole numbers
        n = place[-1] - near if len(place) > near else 0
        while n + 1 < rest and d ** rest * near ** (n + 1) >= far ** (n + 1) * near ** rest:
            n += 1
        place.append(near + n)
    after = [0] * far if causal else [side + b for b in place[1:]]
    return torch.tensor(place[:0:-1] + [0] + after, dtype=torch.int32).to(device)


_FAR = 1024


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


class _Terms:
    """What scores carry besides: checked on their own, and with their problem by :meth:`of`."""

    __slots__ = ("cap", "slopes", "bias", "buckets", "prefix")

    def __init__(self, cap, slopes, bias, buckets, prefix):
        if cap is not None:
            cap = float(cap)
            if not 1e-6 <= cap <= 1024.0:
                raise ValueError(f"a cap must be positive and at most 1024 (got {cap})")
        if (bias is None) != (buckets is None):
            raise ValueError("a bias needs the buckets of its relative positions, and buckets their bias")
        if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("slopes are constants: no gradient is formed of them (pass slopes.detach())")
        self.cap, self.slopes, self.bias, self.buckets, self.prefix = cap, slopes, bias, buckets, prefix

    def of(self, heads: int, segments: int, causal: bool) -> None:
        slopes, bias, buckets, prefix = self.slopes, self.bias, self.buckets, self.prefix
        if slopes is not None:
            if slopes.shape != (heads,) or slopes.dtype != torch.float32:
                raise ValueError(f"slopes must be float32 [{heads}]")
            self.slopes = slopes.contiguous()
        if bias is not None:
            if bias.dim() != 2 or bias.shape[1] != heads or not bias.shape[0] or bias.dtype not in _BIAS:
                raise ValueError(f"the bias must be float32, float16 or bfloat16 [buckets, {heads}]")
            if buckets.dim() != 1 or buckets.dtype != torch.int32 or not buckets.numel() % 2 or buckets.numel() > 2 * _FAR + 1:
                raise ValueError(f"buckets must be int32 [2 far + 1], far at most {_FAR}")
            self.bias, self.buckets = bias.contiguous(), buckets.contiguous()
        if prefix is not None:
            if not causal:
                raise ValueError("a prefix that all queries see belongs to causal segments")
            if prefix.shape != (segments,) or prefix.dtype not in (torch.int32, torch.int64):
                raise ValueError(f"prefix must be int32 [{segments}]")
            if prefix.dtype == torch.int64:  # numbers past 31 bits are as good as the largest one
                prefix = prefix.clamp(0, (1 << 31) - 1).to(torch.int32)
            self.prefix = prefix.contiguous()

    def desc(self) -> _TermsDesc:
        slopes, bias, prefix = _lib.ptr(self.slopes), self.bias, _lib.ptr(self.prefix)
        if bias is None:
            return _TermsDesc(slopes, None, None, prefix, 0, 0, 0, self.cap or 0.0)
        return _TermsDesc(slopes, bias.data_ptr(), self.buckets.data_ptr(), prefix, _lib.DTYPES[bias.dtype], bias.shape[0],
                          self.buckets.numel() // 2, self.cap or 0.0)

    @classmethod
    def again(cls, *values) -> _Terms:
        """Terms that were checked before."""
        t = cls.__new__(cls)
        t.cap, t.slopes, t.bias, t.buckets, t.prefix = values
        return t


_BIAS = (torch.float32, torch.float16, torch.bfloat16)


def _terms(cap, slopes, bias, buckets, prefix=None) -> _Terms | None:
    if cap is None and slopes is None and bias is None and buckets is None and prefix is None:
        return None
    return _Terms(cap, slopes, bias, buckets, prefix)


class _Problem:
    """One checked attention problem: the descriptor and the tensors it points into."""

    terms: _Terms | None = None

    def __init__(self, q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask, terms=None):
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
        if terms is None:
            self.device = _lib.require_gpu(q, k, v, cu_q, cu_k, lens_k, key_mask)
        else:
            terms.of(hq, batch, causal)
            self.device = _lib.require_gpu(q, k, v, cu_q, cu_k, lens_k, key_mask, terms.slopes, terms.bias, terms.buckets,
                                           terms.prefix)
            self.use(terms)
        self.set((q, k, v, cu_q, cu_k, lens_k, key_mask),
                 (total_q, total_k, batch, len_q, len_k, hq, hk, dim, _lib.DTYPES[dtype], 1 if causal else 0, scale))

    @classmethod
    def again(cls, tensors, sizes, terms=None) -> _Problem:
        """A problem that was checked before, of its ``tensors`` (or copies of them) and ``sizes``."""
        p = cls.__new__(cls)
        p.device = tensors[0].device
        if terms is not None:
            p.use(terms)
        p.set(tensors, sizes)
        return p

    def use(self, terms: _Terms) -> None:
        self.terms, self.terms_desc = terms, terms.desc()
        self.terms_ref = ctypes.byref(self.terms_desc)

    def set(self, tensors, sizes) -> None:
        (q, q_s), (k, k_s), (v, v_s) = _heads(tensors[0]), _heads(tensors[1]), _heads(tensors[2])
        self.tensors, self.sizes = (q, k, v, *tensors[3:]), sizes
        strides = (0, *q_s[:2], 0, *k_s[:2], 0, *v_s[:2]) if len(q_s) == 3 else (*q_s[:3], *k_s[:3], *v_s[:3])
        self.desc = _Desc(*[x if x is None else x.data_ptr() for x in self.tensors], strides, *sizes)
        self.ref = ctypes.byref(self.desc)

    def forward(self, want_lse: bool, want_rest: bool = False) -> tuple[torch.Tensor, ...]:
        """``out`` and ``lse``; with ``want_rest`` and terms also what rounding took from ``out``, where it is kept."""
        q, ref = self.tensors[0], self.ref
        out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=self.device) if want_lse else None
        if self.terms is None:
            need = _lib.query("hi3d_attention_workspace", ref)
            work = _lib.workspace(need, self.device) if need else None
            _lib.call("hi3d_attention_forward", ref, out.data_ptr(), _lib.ptr(lse), _lib.ptr(work), need,
                      _lib.stream(self.device))
            return out, lse
        kept = ctypes.c_int32(0) if want_rest else None
        need = _lib.query("hi3d_attention_terms_workspace", ref, self.terms_ref, kept if kept is None else ctypes.byref(kept))
        work = _lib.workspace(need, self.device) if need else None
        rest = torch.empty_like(out) if want_rest and kept.value else None
        _lib.call("hi3d_attention_terms_forward", ref, self.terms_ref, out.data_ptr(), _lib.ptr(rest), _lib.ptr(lse),
                  _lib.ptr(work), need, _lib.stream(self.device))
        return (out, lse, rest) if want_rest else (out, lse)

    def backward(self, out, lse, dout, dlse, want_q: bool, want_kv: bool, want_bias: bool = False, rest=None):
        q, k = self.tensors[:2]
        if (q.shape[-2] // k.shape[-2] - 1) * q.stride(-2) >= 1 << 29:  # a tile's queries are addressed with 32 bits
            self.set((q.contiguous(), *self.tensors[1:]), self.sizes)
        ref = self.ref
        out, lse, dout = _dense(out), _dense(lse), _dense(dout)
        dlse = dlse if dlse is None else _dense(dlse)
        dq = torch.empty(q.shape, dtype=q.dtype, device=self.device) if want_q else None
        dk = torch.empty(k.shape, dtype=k.dtype, device=self.device) if want_kv else None
        dv = torch.empty(k.shape, dtype=k.dtype, device=self.device) if want_kv else None
        if self.terms is None:
            need = _lib.query("hi3d_attention_backward_workspace", ref)
            work = _lib.workspace(need, self.device) if need else None
            _lib.call("hi3d_attention_backward", ref, out.data_ptr(), lse.data_ptr(), dout.data_ptr(),
                      _lib.ptr(dlse), _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv), _lib.ptr(work), need, _lib.stream(self.device))
            return dq, dk, dv, None
        dbias = torch.empty_like(self.terms.bias) if want_bias else None
        need = _lib.query("hi3d_attention_terms_backward_workspace", ref, self.terms_ref)
        work = _lib.workspace(need, self.device) if need else None
        _lib.call("hi3d_attention_terms_backward", ref, self.terms_ref, out.data_ptr(), _lib.ptr(rest), lse.data_ptr(),
                  dout.data_ptr(), _lib.ptr(dlse), _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv), _lib.ptr(dbias), _lib.ptr(work),
                  need, _lib.stream(self.device))
        return dq, dk, dv, dbias


def _dense(x: torch.Tensor) -> torch.Tensor:
    x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, cu_q, cu_k, lens_k, scale, causal, key_mask, terms):
        p = _Problem(q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask, terms)
        ctx.sizes, ctx.with_terms = p.sizes, terms is not None
        with _lib.on(p.device):
            if terms is None:
                out, lse = p.forward(True)
                ctx.save_for_backward(*p.tensors, out, lse)
            else:
                ctx.cap = terms.cap
                out, lse, rest = p.forward(True, True)
                ctx.save_for_backward(*p.tensors, out, lse, rest, terms.slopes, terms.bias, terms.buckets, terms.prefix)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    def backward(ctx, dout, dlse):
        if torch.is_grad_enabled():
            raise RuntimeError("attention is differentiable once")
        needs = ctx.needs_input_grad
        want_q, want_kv, want_bias = needs[0], needs[1] or needs[2], needs[3]
        if (dout is None and dlse is None) or not (want_q or want_kv or want_bias):
            return (None,) * 11
        saved = ctx.saved_tensors
        tensors, out, lse, rest, terms = saved[:7], saved[7], saved[8], None, None
        if ctx.with_terms:
            rest, terms = saved[9], _Terms.again(ctx.cap, *saved[10:])
        dout = torch.zeros_like(out) if dout is None else dout
        p = _Problem.again(tensors, ctx.sizes, terms)
        with _lib.on(p.device):
            dq, dk, dv, dbias = p.backward(out, lse, dout, dlse, want_q, want_kv, want_bias, rest)
        return dq, dk, dv, dbias, None, None, None, None, None, None, None


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
    cap: float | None = None,
    slopes: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    buckets: torch.Tensor | None = None,
    prefix: torch.Tensor | None = None,
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

    Scores may carry terms. With ``x = scale * q k`` and ``r = j - (i + lk - lq)``, the place of
    key ``j`` relative to query ``i`` (the last of ``lq`` queries stands at the last of ``lk`` keys):

    * ``cap`` (at most 1024): ``cap * tanh(x / cap)`` in place of ``x``;
    * ``slopes`` (float32 ``[hq]``, constants, as of :func:`head_slopes`): less ``slopes[h] * |r|``. A row whose
      largest score is below -2.9e6, past which fp32 has no digits for it, counts as one that sees no key;
    * ``bias`` (``[count, hq]``, float32, fp16 or bf16) with ``buckets`` (int32 ``[2 far + 1]``, far at
      most 1024, as of :func:`relative_buckets`): plus ``bias[buckets[clamp(r, -far, far) + far], h]``.
      Differentiable in ``bias``. A bias below -1e5 hides its keys; a bucket outside the table
      counts as the nearest one;
    * ``prefix`` (int32, one per segment), with ``causal``: keys ``j < prefix`` are seen by every query.

    Returns ``[..., hq, dim]`` (and with ``return_lse`` the float32 ``log(sum(exp(scores)))``
    per row and head, -inf for a row that sees no key). Differentiable once in ``q``, ``k``, ``v``
    and ``bias`` (reverse mode), through both outputs; :func:`attend_grad` is the same without autograd
    (and says for which values fp16 gradients are formed)."""
    _lib.no_tangents("attention", q, k, v, slopes, bias)
    terms = _terms(cap, slopes, bias, buckets, prefix)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or
                                    (bias is not None and bias.requires_grad)):
        out, lse = _Attend.apply(q, k, v, bias, cu_q, cu_k, lens_k, scale, causal, key_mask, terms)
        return (out, lse) if return_lse else out
    p = _Problem(q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask, terms)
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
    cap: float | None = None,
    slopes: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    buckets: torch.Tensor | None = None,
    prefix: torch.Tensor | None = None,
) -> tuple[torch.Tensor, ...]:
    """``dq``, ``dk`` and ``dv`` (and ``dbias``, where there is a bias) of :func:`attend` from its
    arguments, its ``out`` and ``lse``, the gradient ``dout`` of ``out`` and optionally ``dlse`` of ``lse``.
    (With terms autograd keeps more digits of ``out`` than its type holds; from ``out`` alone this
    walks over the keys once more for them.)

    Sums run in a fixed order: the same bits every time. fp32 sums; probabilities and score
    gradients are rounded once to the inputs' type for their products (in fp16 after a scaling
    by powers of two, so that small gradients of long rows keep their digits; with values of 8190
    and more that scaling can leave fp16's range, and the gradients of such a row are not finite
    then: take bf16 there). Launches only:
    this is the form to capture into a graph, with no autograd node of another stream in it."""
    _lib.no_tangents("attention", q, k, v, out, lse, dout, dlse, slopes, bias)
    terms = _terms(cap, slopes, bias, buckets, prefix)
    p = _Problem(q, k, v, cu_q, cu_k, lens_k, scale, causal, key_mask, terms)
    for name, x, shape, dtype in (("out", out, q.shape, q.dtype), ("dout", dout, q.shape, q.dtype),
                                  ("lse", lse, q.shape[:-1], torch.float32), ("dlse", dlse, q.shape[:-1], torch.float32)):
        if x is not None and (x.shape != shape or x.dtype != dtype):
            raise ValueError(f"{name} must be {list(shape)} of {dtype} (got {list(x.shape)} of {x.dtype})")
    _lib.require_gpu(q, out, lse, dout, dlse)
    with _lib.on(p.device), torch.no_grad():
        grads = p.backward(out, lse, dout, dlse, True, True, bias is not None)
    return grads if bias is not None else grads[:3]


def attend_shared(
    q: torch.Tensor,
    shared_k: torch.Tensor,
    shared_v: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    lens_k: torch.Tensor | None = None,
    scale: float | None = None,
    causal: bool = False,
    shared_mask: torch.Tensor | None = None,
    key_mask: torch.Tensor | None = None,
    return_lse: bool = False,
    cap: float | None = None,
    slopes: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    buckets: torch.Tensor | None = None,
):
    """:func:`attend` of ``q [B, L, hq, dim]`` over keys that all ``B`` sequences share, ``shared_k`` and
    ``shared_v [P, hk, dim]``, and behind them each sequence's own, ``k`` and ``v [B, M, hk, dim]`` with
    ``lens_k [B]`` of them in use. The shared keys are read once for the batch.

    ``causal`` limits the own keys (query ``i`` of ``L`` sees ``j <= i + lens_k - L``); every query sees
    the shared ones, but those where ``shared_mask [P]`` is False. Positions relative to a query, for
    ``slopes`` and ``bias``, go through the shared keys to the own ones without a gap. For serving: no
    gradients are formed."""
    _lib.no_tangents("attention", q, shared_k, shared_v, k, v, slopes, bias)
    given = (q, shared_k, shared_v, k, v, bias)
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in given):
        raise NotImplementedError("attention over shared keys forms no gradients (concatenate the keys for attend)")
    if q.dim() != 4:
        raise ValueError("q must be [batch, length, heads, dim]")
    p = _Problem(q, k, v, None, None, lens_k, scale, causal, key_mask, _Terms(cap, slopes, bias, buckets, None))
    for name, x in (("shared_k", shared_k), ("shared_v", shared_v)):
        if x.dim() != 3 or x.shape[1:] != k.shape[2:] or x.dtype != q.dtype:
            raise ValueError(f"{name} must be [keys, {k.shape[2]}, {k.shape[3]}] of {q.dtype}")
    if shared_k.shape[0] + k.shape[1] >= (1 << 31) - 64:
        raise ValueError("shared and own keys of a sequence must be fewer than 2^31 - 64")
    if shared_k.shape != shared_v.shape:
        raise ValueError(f"keys {list(shared_k.shape)} and values {list(shared_v.shape)} differ")
    if shared_mask is not None:
        if shared_mask.dtype not in (torch.bool, torch.uint8) or shared_mask.shape != shared_k.shape[:1]:
            raise ValueError(f"shared_mask must be bool [{shared_k.shape[0]}]")
        shared_mask = shared_mask.contiguous()
    device = _lib.require_gpu(q, shared_k, shared_v, shared_mask)
    (shared_k, ks), (shared_v, vs) = _heads(shared_k), _heads(shared_v)
    shared = _SharedDesc(shared_k.data_ptr(), shared_v.data_ptr(), _lib.ptr(shared_mask), (*ks[:2], *vs[:2]), shared_k.shape[0])
    ref = ctypes.byref(shared)
    with _lib.on(device):
        q = p.tensors[0]
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
        lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=device) if return_lse else None
        need = _lib.query("hi3d_attention_shared_workspace", p.ref, p.terms_ref, ref)
        work = _lib.workspace(need, device) if need else None
        _lib.call("hi3d_attention_shared_forward", p.ref, p.terms_ref, ref, out.data_ptr(), _lib.ptr(lse), _lib.ptr(work),
                  need, _lib.stream(device))
    return (out, lse) if return_lse else out
