"""What attention with terms refuses because its numbers would leave their types. No GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from test_attention_terms_host import _desc


@pytest.mark.parametrize("shared,own,fits", [
    ((1 << 31) - 1, 100, False), ((1 << 31) - 100, 36, False), (1000, (1 << 31) - 900, False),
    ((1 << 31) - 200, 100, True), (1 << 30, 1 << 20, True)])
def test_places_over_shared_and_own_keys_fit_31_bits(shared, own, fits, monkeypatch):
    from hi3d_amd import _lib, attention

    d, t, out = _desc(attention, nq=1, nk=own), attention._TermsDesc(), ctypes.c_int64(7)
    s = attention._SharedDesc(4096, 4096, None, (128, 64, 128, 64), shared)
    args = (ctypes.byref(d), ctypes.byref(t), ctypes.byref(s), ctypes.byref(out))
    if fits:
        _lib.call("hi3d_attention_shared_workspace", *args)
        return
    with pytest.raises(ValueError, match="2\\^31"):
        _lib.call("hi3d_attention_shared_workspace", *args)
    monkeypatch.setattr(_lib, "require_gpu", lambda *x: torch.device("cpu"))  # the checks behind it are this test's
    one = torch.zeros(1, 2, 64).half()
    keys, cache = one.expand(shared, 2, 64), one[None].expand(1, own, 2, 64)
    with pytest.raises(ValueError, match="2\\^31"):
        attention.attend_shared(torch.zeros(1, 1, 4, 64).half(), keys, keys, cache, cache)


@pytest.mark.parametrize("scale,cap,fits", [(1e33, 1e-6, False), (3e38, 1.0, False), (1e30, 1e-6, True), (1e38, 30.0, True)])
def test_scores_over_the_cap_are_numbers(scale, cap, fits):
    """Infinite, and a score of zero over it is none."""
    from hi3d_amd import _lib, attention

    d, t, out = _desc(attention, scale=scale), attention._TermsDesc(cap=cap), ctypes.c_int64(7)
    for name, more in (("hi3d_attention_terms_workspace", (None,)), ("hi3d_attention_terms_backward_workspace", ())):
        args = (ctypes.byref(d), ctypes.byref(t), *more, ctypes.byref(out))
        if fits:
            _lib.call(name, *args)
        else:
            with pytest.raises(ValueError, match="scale / cap"):
                _lib.call(name, *args)
