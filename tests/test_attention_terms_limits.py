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
