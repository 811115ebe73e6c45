"""Derivatives that the token operators do not have are refused, not dropped."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad


@pytest.mark.parametrize("which", [0, 1, 2])
def test_attention_refuses_tangents(which):
    from hi3d_amd import attention

    qkv = [torch.randn(4, 2, 64).half() for _ in range(3)]
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="ROCm GPU only"):  # no tangent: the usual refusal of host tensors
            attention.attend(*qkv)
        qkv[which] = forward_ad.make_dual(qkv[which], torch.ones_like(qkv[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            attention.attend(*qkv)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            attention.attend(*qkv)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            attention.attend_grad(*qkv, qkv[0], torch.zeros(4, 2), qkv[0])


@pytest.mark.parametrize("which", range(3))
def test_attention_gradients_refuse_tangents(which):
    from hi3d_amd import attention

    q = torch.randn(4, 2, 64).half()
    rest = [q, torch.zeros(4, 2), q]
    with forward_ad.dual_level():
        rest[which] = forward_ad.make_dual(rest[which], torch.ones_like(rest[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            attention.attend_grad(q, q, q, *rest)


def test_rotary_refuses_tangents():
    from hi3d_amd import rotary

    x, p, f = torch.randn(4, 2, 64), torch.zeros(4, 1, dtype=torch.int32), rotary.frequencies(64)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="ROCm GPU only"):
            rotary.rotate(x, p, f)
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: rotary.rotate(dual, p, f), lambda: rotary.rotate_qk(x, dual, p, f),
                     lambda: rotary.rotate(x, p, forward_ad.make_dual(f, torch.ones_like(f)))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_rotary_refuses_gradients_of_frequencies():
    """Frequencies are constants: a leaf that waits for their gradient would get none."""
    from hi3d_amd import rotary

    x, p, f = torch.randn(4, 2, 64), torch.zeros(4, 1, dtype=torch.int32), rotary.frequencies(64).requires_grad_(True)
    for call in (lambda: rotary.rotate(x, p, f), lambda: rotary.rotate(x.requires_grad_(True), p, f)):
        with pytest.raises(NotImplementedError, match="frequencies"):
            call()
    with torch.no_grad(), pytest.raises(ValueError, match="ROCm GPU only"):
        rotary.rotate(x, p, f)
