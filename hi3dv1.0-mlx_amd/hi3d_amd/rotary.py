"""Rotary positions of token heads, with gradients.

Pair ``p`` of every head of a token turns by ``t = sum_a positions[token, a] *
freqs[a, p]``: one axis for sequences, three for voxels (:func:`frequencies` gives each
axis its own pairs, and stretched positions for contexts longer than the trained one). The
angle is formed and reduced in float64 on the GPU, so far positions keep their digits.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

_POSITIONS = {torch.int32: _lib.I32, torch.int64: _lib.I64}


def frequencies(
    rot: int,
    *,
    axes: int = 1,
    base: float = 10000.0,
    stretch: float = 1.0,
    scaling: str = "linear",
    trained: int = 0,
    device: torch.device | str | None = None,
) -> torch.Tensor:
    """``freqs [axes, rot / 2]`` (float64): axis ``a`` owns pairs ``a * m .. a * m + m - 1``
    with ``m = rot / 2 // axes`` and frequencies ``base ** (-i / m)``; left-over pairs stay as
    they are.

    ``stretch`` > 1 fits positions past the trained length. ``scaling`` says how:
    ``"linear"`` (position interpolation, Chen et al., 2023) divides every frequency by it;
    ``"base"`` (the "NTK-aware" change of base) raises the base to ``base * stretch ** (m / (m -
    1))``, which leaves the fastest pair and divides the slowest by ``stretch``; ``"blend"``
    (by parts, as in YaRN, Peng et al., 2023, without its temperature) leaves pairs that turn 32
    times or more within ``trained`` positions, divides those that turn once or less, and goes
    between by the number of turns.
    """
    if rot < 0 or rot % 2:
        raise ValueError(f"the number of turned values must be even (got {rot})")
    if not 1 <= axes <= 4:
        raise ValueError(f"1 to 4 position axes (got {axes})")
    if scaling not in ("linear", "base", "blend"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if not (stretch >= 1.0 and math.isfinite(stretch) and base > 1.0 and math.isfinite(base)):
        raise ValueError("stretch must be at least 1 and base above 1")
    m = rot // 2 // axes
    i = torch.arange(m, dtype=torch.float64)
    if scaling == "base" and m > 1:
        f = (base * stretch ** (m / (m - 1))) ** (-i / m)
    else:
        f = base ** (-i / max(m, 1))
        if scaling == "blend":
            if trained <= 0:
                raise ValueError("blend scaling needs the trained length")
            keep = ((trained * f / (2 * math.pi) - 1) / 31).clamp(0.0, 1.0)
            f = f * keep + f / stretch * (1 - keep)
        else:
            f = f / stretch
    freqs = torch.zeros((axes, rot // 2), dtype=torch.float64)
    for a in range(axes):
        freqs[a, a * m:(a + 1) * m] = f
    return freqs.to(device) if device is not None else freqs


def _tokens(x: torch.Tensor, what: str) -> torch.Tensor:
    """``[..., H, D]`` as rows of heads ``[N, H, D]`` with adjacent values."""
    if x.dim() < 3:
        raise ValueError(f"{what} must be [..., heads, dim]")
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        x = x.contiguous()
    return x.reshape(-1, *x.shape[-2:]) if x.dim() > 3 else x


_Two, _TwoHeads, _FourStrides = ctypes.c_void_p * 2, ctypes.c_int32 * 2, ctypes.c_int64 * 4


def _launch(xs, positions: torch.Tensor, freqs: torch.Tensor, interleaved: bool, scale: float,
            inverse: bool) -> list[torch.Tensor]:
    flat = [_tokens(x, "x") for x in xs]
    a, b = flat[0], flat[-1]
    n, heads, dim = a.shape
    a_s, b_s, axes = a.stride(), b.stride(), freqs.shape[0]
    pos = positions if positions.shape == (n, axes) else positions.reshape(n, axes)
    device, dtype = a.device, a.dtype
    outs = [torch.empty(x.shape, dtype=dtype, device=device) for x in xs]
    one = len(xs) == 1
    _lib.call(
        "hi3d_rotary", _Two(a.data_ptr(), None if one else b.data_ptr()),
        _Two(outs[0].data_ptr(), None if one else outs[1].data_ptr()), _TwoHeads(heads, 0 if one else b.shape[1]),
        _FourStrides(a_s[0], a_s[1], b_s[0], b_s[1]), _lib.DTYPES[dtype], n, dim, 2 * freqs.shape[1], pos.data_ptr(),
        _POSITIONS[pos.dtype], pos.stride(0), pos.stride(1), axes, freqs.data_ptr(), interleaved, inverse, scale,
        _lib.stream(device),
    )
    return outs


class _Rotate(torch.autograd.Function):
    """A rotation's gradient is the opposite rotation, so it can be differentiated again."""

    @staticmethod
    def forward(ctx, positions, freqs, interleaved, scale, inverse, *xs):
        ctx.save_for_backward(positions, freqs)
        ctx.how = (interleaved, scale, inverse)
        ctx.set_materialize_grads(False)
        with _lib.on(xs[0].device):
            return tuple(_launch(xs, positions, freqs, interleaved, scale, inverse))

    @staticmethod
    def backward(ctx, *grads):
        positions, freqs = ctx.saved_tensors
        interleaved, scale, inverse = ctx.how
        out: list[torch.Tensor | None] = [None] * len(grads)
        given = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[5 + i]]
        if given:
            way = (positions, freqs, interleaved, scale, not inverse)
            if torch.is_grad_enabled():
                back = _Rotate.apply(*way, *[grads[i] for i in given])
            else:
                with _lib.on(positions.device):
                    back = _launch([grads[i] for i in given], *way)
            for i, g in zip(given, back):
                out[i] = g
        return (None, None, None, None, None, *out)


def _rotate(xs: list[torch.Tensor], positions: torch.Tensor, freqs: torch.Tensor, layout: str, scale: float):
    if layout not in ("half", "interleaved"):
        raise ValueError(f"unknown layout {layout!r}")
    lead, dim, dtype = xs[0].shape[:-2], xs[0].shape[-1] if xs[0].dim() else 0, xs[0].dtype
    for x in xs:
        if x.dim() < 3 or x.shape[:-2] != lead or x.shape[-1] != dim:
            raise ValueError("queries and keys must be [..., heads, dim] of the same tokens and head size")
        if x.dtype != dtype:
            raise ValueError(f"queries and keys of different types: {dtype} and {x.dtype}")
    if dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"unsupported dtype {dtype}")
    if freqs.dim() != 2 or freqs.dtype != torch.float64:
        raise ValueError("freqs must be float64 [axes, rot / 2]")
    if 2 * freqs.shape[1] > dim:
        raise ValueError(f"freqs turn {2 * freqs.shape[1]} values of heads of {dim}")
    if positions.dtype not in _POSITIONS:
        raise ValueError("positions must be int32 or int64")
    if positions.shape != (*lead, freqs.shape[0]) and not (freqs.shape[0] == 1 and positions.shape == lead):
        raise ValueError(f"positions must be {[*lead, int(freqs.shape[0])]} (got {list(positions.shape)})")
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if freqs.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("frequencies are constants: no gradient is formed of them (pass freqs.detach())")
    _lib.no_tangents("rotary", *xs, freqs)
    _lib.require_gpu(*xs, positions, freqs)
    freqs = freqs.contiguous()
    if torch.is_grad_enabled() and any(x.requires_grad for x in xs):
        return _Rotate.apply(positions, freqs, layout == "interleaved", float(scale), False, *xs)
    with _lib.on(xs[0].device):
        return _launch(xs, positions, freqs, layout == "interleaved", float(scale), False)


def rotate(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, *, layout: str = "half",
           scale: float = 1.0) -> torch.Tensor:
    """``x [..., heads, dim]`` (fp32, fp16 or bf16) with the first ``2 * freqs.shape[1]`` values
    of every head turned by ``positions [..., axes]`` (int32 or int64; ``[...]`` for one axis)
    and multiplied by ``scale``; the rest is copied. Pairs are ``(p, p + rot / 2)``
    (``layout="half"``) or ``(2 p, 2 p + 1)`` (``"interleaved"``). fp32 arithmetic, one
    rounding; differentiable (reverse mode)."""
    return _rotate([x], positions, freqs, layout, scale)[0]


def rotate_qk(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, *, layout: str = "half",
              scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`rotate` of queries and keys of the same tokens in one launch (their numbers of
    heads may differ, and they may be views of one projection)."""
    a, b = _rotate([q, k], positions, freqs, layout, scale)
    return a, b
