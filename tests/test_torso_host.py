"""The torso's token operators without a GPU: their float64 oracles against closed forms and
other formulas, and the refusals of the Python and C entry points."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import attention as oattention
from oracle import rotary as orotary


# ------------------------------------------------------------------------ oracles


def test_attention_oracle_closed_forms():
    rng = np.random.default_rng(0)
    v = rng.standard_normal((6, 2, 8))
    r = oattention.forward(np.zeros((3, 4, 8)), np.zeros((6, 2, 8)), v, [(0, 3)], [(0, 6)])
    assert np.allclose(r["out"], np.repeat(v.mean(0), 2, 0)[None]) and np.allclose(r["lse"], math.log(6))
    r = oattention.forward(np.zeros((3, 2, 8)), np.zeros((6, 2, 8)), v, [(0, 3)], [(0, 6)], causal=True)
    for i in range(3):
        assert np.allclose(r["out"][i], v[:i + 4].mean(0))
    r = oattention.forward(np.zeros((4, 2, 8)), np.zeros((2, 2, 8)), v[:2], [(0, 4)], [(0, 2)], causal=True)
    assert not r["out"][:2].any() and np.isneginf(r["lse"][:2]).all() and np.allclose(r["out"][2], v[0])


def test_attention_oracle_gradients_against_torch():
    rng = np.random.default_rng(1)
    q, k, v, do = rng.standard_normal((5, 4, 8)), rng.standard_normal((7, 2, 8)), rng.standard_normal((7, 2, 8)), rng.standard_normal((5, 4, 8))
    r = oattention.backward(q, k, v, do, [(0, 5)], [(0, 7)], causal=True)
    tq, tk, tv = (torch.tensor(x, requires_grad=True) for x in (q, k, v))
    s = torch.einsum("ihd,jhd->hij", tq, tk.repeat_interleave(2, 1)) * 8 ** -0.5
    s = s.masked_fill(torch.arange(7) > torch.arange(5)[:, None] + 2, -math.inf)
    out = torch.einsum("hij,jhd->ihd", s.softmax(-1), tv.repeat_interleave(2, 1))
    out.backward(torch.tensor(do))
    for name, t in (("dq", tq), ("dk", tk), ("dv", tv)):
        assert np.allclose(r[name], t.grad.numpy())


def test_rotary_oracle():
    x = np.zeros((1, 1, 4))
    x[0, 0, 0] = 1.0
    y = orotary.rotate(x, [[1]], np.array([[math.pi / 2, 0.0]]))
    assert np.allclose(y[0, 0], [0, 0, 1, 0])
    y = orotary.rotate(x, [[1]], np.array([[math.pi / 2, 0.0]]), "interleaved", 2.0)
    assert np.allclose(y[0, 0], [0, 2, 0, 0])
    rng = np.random.default_rng(2)
    x, p, f = rng.standard_normal((5, 2, 12)), rng.integers(0, 99, (5, 3)), rng.random((3, 4))
    y = orotary.rotate(x, p, f)
    assert np.allclose(orotary.rotate(y, p, f, inverse=True), x)
    assert np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1)) and np.array_equal(y[..., 8:], x[..., 8:])


# -------------------------------------------------------------------- frequencies


def test_frequencies():
    from hi3d_amd import rotary

    f = rotary.frequencies(64)
    assert f.shape == (1, 32) and f.dtype == torch.float64 and f[0, 0] == 1.0
    assert torch.allclose(f[0], 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32), rtol=1e-14)
    f3 = rotary.frequencies(64, axes=3)
    assert f3.shape == (3, 32) and int((f3 != 0).sum()) == 30 and not f3[:, 30:].any()
    for a in range(3):
        assert torch.equal(f3[a, 10 * a:10 * a + 10], f3[0, :10])
    assert torch.allclose(rotary.frequencies(64, stretch=4.0), f / 4, rtol=1e-14)
    b = rotary.frequencies(64, stretch=4.0, scaling="base")
    assert b[0, 0] == 1.0 and abs(float(b[0, -1] / f[0, -1]) - 0.25) < 1e-12
    m = rotary.frequencies(64, stretch=4.0, scaling="blend", trained=4096)
    turns = 4096 * f[0] / (2 * math.pi)
    assert torch.equal(m[0][turns >= 32], f[0][turns >= 32])
    assert torch.allclose(m[0][turns <= 1], f[0][turns <= 1] / 4, rtol=1e-14)
    middle = (turns > 1) & (turns < 32)
    assert bool(middle.any()) and bool((m[0][middle] < f[0][middle]).all()) and bool((m[0][middle] > f[0][middle] / 4).all())
    assert rotary.frequencies(0).shape == (1, 0)
    for bad in (dict(rot=3), dict(rot=-2), dict(rot=8, axes=5), dict(rot=8, axes=0), dict(rot=8, stretch=0.5),
                dict(rot=8, stretch=math.nan), dict(rot=8, base=1.0), dict(rot=8, scaling="x"),
                dict(rot=8, scaling="blend")):
        with pytest.raises(ValueError):
            rotary.frequencies(**bad)


# ----------------------------------------------------------------------- refusals


def test_rotary_refusals():
    from hi3d_amd import rotary

    x, p, f = torch.zeros(4, 2, 64), torch.zeros(4, 3, dtype=torch.int32), rotary.frequencies(64, axes=3)
    with pytest.raises(ValueError, match="ROCm GPU only"):
        rotary.rotate(x, p, f)
    for match, args, kw in [
        ("layout", (x, p, f), dict(layout="x")), ("heads, dim", (x[0], p, f), {}), ("dtype", (x.double(), p, f), {}),
        ("float64", (x, p, f.float()), {}), ("float64", (x, p, f[0]), {}), ("int32 or int64", (x, p.float(), f), {}),
        ("positions must be", (x, p[:, :2], f), {}), ("positions must be", (x, p[:3], f), {}),
        ("positions must be", (x, p[:, 0], f), {}), ("heads of 62", (x[..., :62], p, f), {}),
        ("finite", (x, p, f), dict(scale=math.inf))]:
        with pytest.raises(ValueError, match=match):
            rotary.rotate(*args, **kw)
    for k in (x[:3], x.half(), x[..., :32]):
        with pytest.raises(ValueError):
            rotary.rotate_qk(x, k, p, f)


def test_rotary_c_refusals():
    from hi3d_amd import _lib

    buf = ctypes.create_string_buffer(64)
    at = ctypes.addressof(buf)

    def call(**kw):
        a = dict(x=(ctypes.c_void_p * 2)(at, None), y=(ctypes.c_void_p * 2)(at, None), heads=(ctypes.c_int32 * 2)(1, 0),
                 strides=(ctypes.c_int64 * 4)(8, 8, 0, 0), dtype=_lib.F32, n=1, dim=8, rot=8, pos=at, ptype=_lib.I32,
                 prow=1, paxis=1, axes=1, freqs=at, inter=0, inv=0, scale=1.0, stream=None)
        a.update(kw)
        _lib.call("hi3d_rotary", *a.values())

    call(n=0)
    call(heads=(ctypes.c_int32 * 2)(0, 0))
    for match, kw in [("type 3", dict(dtype=_lib.F64)), ("int32 or int64", dict(ptype=_lib.F32)), ("bad sizes", dict(n=-1)),
                      ("bad sizes", dict(heads=(ctypes.c_int32 * 2)(-1, 0))), ("head size", dict(dim=0)),
                      ("head size", dict(dim=1025)), ("turned values", dict(rot=7)), ("turned values", dict(rot=10)),
                      ("axes", dict(axes=0)), ("axes", dict(axes=5)), ("null", dict(pos=None)), ("null", dict(freqs=None)),
                      ("null", dict(x=(ctypes.c_void_p * 2)(None, None))), ("null", dict(x=None))]:
        with pytest.raises(ValueError, match=match):
            call(**kw)


def _qkv(n=4, hq=2, hk=2, d=64, dtype=torch.float16):
    return torch.zeros(n, hq, d, dtype=dtype), torch.zeros(n, hk, d, dtype=dtype), torch.zeros(n, hk, d, dtype=dtype)


def test_attention_refusals():
    from hi3d_amd import attention

    q, k, v = _qkv()
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm GPU only"):
        attention.attend(q, k, v)
    dense = [x[None] for x in (q, k, v)]
    for match, args, kw in [
        ("fp16 or bf16", _qkv(dtype=torch.float32), {}), ("multiple of 8", _qkv(d=60), {}), ("multiple of 8", _qkv(d=136), {}),
        ("multiple of 8", _qkv(d=0), {}), ("no multiple", _qkv(hq=3, hk=2), {}), ("no multiple", _qkv(hk=0), {}),
        ("different types", (q, k.bfloat16(), v), {}), ("keys .* and values", (q, k, v[:3]), {}),
        ("heads of", (q, k[..., :32], v[..., :32]), {}), ("must be \\[tokens", (q[0], k[0], v[0]), {}),
        ("must be \\[tokens", (q, k[None], v[None]), {}), ("int32 offsets", (q, k, v, cu.float()), {}),
        ("int32 offsets", (q, k, v, cu[None]), {}), ("int32 offsets", (q, k, v, cu[:0]), {}),
        ("same segments", (q, k, v, cu, torch.tensor([0, 2, 4], dtype=torch.int32)), {}),
        ("same segments", (q, k, v, None, cu), {}), ("offsets of their own", (q[:3], k, v, cu), {}),
        ("without a segment", (q, k, v, cu[:1]), {}), ("packed tokens", (*dense, cu), {}),
        ("batch elements", (dense[0], dense[1].expand(2, -1, -1, -1), dense[2].expand(2, -1, -1, -1)), {}),
        ("lens_k", (q, k, v), dict(lens_k=cu[:1])), ("lens_k", tuple(dense), dict(lens_k=cu)),
        ("key_mask", (q, k, v), dict(key_mask=torch.ones(3, dtype=torch.bool))),
        ("key_mask", (q, k, v), dict(key_mask=torch.ones(4))), ("scale", (q, k, v), dict(scale=0.0)),
        ("scale", (q, k, v), dict(scale=-1.0)), ("scale", (q, k, v), dict(scale=math.nan))]:
        with pytest.raises(ValueError, match=match):
            attention.attend(*args, **kw)
    with pytest.raises(ValueError, match="segment of -1"):
        attention.offsets([3, -1], "cpu")
    with pytest.raises(ValueError, match="31 bits"):
        attention.offsets([1 << 30, 1 << 30], "cpu")
    assert attention.offsets([3, 0, 2], "cpu").tolist() == [0, 3, 3, 5]


def _desc(**kw):
    from hi3d_amd import _lib, attention

    d = attention._Desc()
    d.q = d.k = d.v = 4096
    d.total_q = d.total_k = d.len_q = d.len_k = 4
    d.batch, d.heads_q, d.heads_k, d.dim, d.dtype, d.scale = 1, 4, 2, 64, _lib.F16, 0.125
    d.strides[:] = [0, 256, 64, 0, 128, 64, 0, 128, 64]
    for name, value in kw.items():
        if name.startswith("stride"):
            d.strides[int(name[6:])] = value
        else:
            setattr(d, name, value)
    return d


def test_attention_c_refusals():
    from hi3d_amd import _lib

    query = lambda **kw: _lib.query("hi3d_attention_workspace", ctypes.byref(_desc(**kw)))  # noqa: E731
    assert query() == 0
    assert query(len_k=65536, total_k=65536, total_q=1, len_q=1) > 0
    for match, kw in [("type 0", dict(dtype=_lib.F32)), ("head size", dict(dim=4)), ("head size", dict(dim=136)),
                      ("no multiple", dict(heads_q=3)), ("no multiple", dict(heads_k=0)), ("bad sizes", dict(batch=-1)),
                      ("not 1 segments", dict(len_q=3)), ("not 1 segments", dict(len_k=5)), ("scale", dict(scale=0.0)),
                      ("scale", dict(scale=math.inf)), ("scale", dict(scale=math.nan)), ("aligned", dict(q=4098)),
                      ("multiples of 8", dict(stride2=60)), ("multiples of 8", dict(stride4=129)),
                      ("row strides", dict(stride1=1 << 23)), ("row strides", dict(stride7=-128)),
                      ("null", dict(q=None)), ("null", dict(v=None)), ("lens_k", dict(lens_k=64, cu_k=64)),
                      ("2\\^31", dict(total_q=1 << 31, cu_q=64)), ("too many rows", dict(total_q=(1 << 30), cu_q=64))]:
        with pytest.raises(ValueError, match=match):
            query(**kw)
    with pytest.raises(ValueError, match="null"):
        _lib.query("hi3d_attention_workspace", None)
    with pytest.raises(ValueError, match="without a segment"):
        _lib.call("hi3d_attention_forward", ctypes.byref(_desc(batch=0, cu_q=64, cu_k=64)), 4096, None, None, 0, None)
    with pytest.raises(ValueError, match="out must be"):
        _lib.call("hi3d_attention_forward", ctypes.byref(_desc()), None, None, None, 0, None)


def test_attention_oracle_gradient_of_lse():
    rng = np.random.default_rng(2)
    q, k, v = rng.standard_normal((5, 4, 8)), rng.standard_normal((7, 2, 8)), rng.standard_normal((7, 2, 8))
    do, dl = rng.standard_normal((5, 4, 8)), rng.standard_normal((5, 4))
    r = oattention.backward(q, k, v, do, [(0, 5)], [(0, 7)], dlse=dl)
    tq, tk, tv = (torch.tensor(x, requires_grad=True) for x in (q, k, v))
    s = torch.einsum("ihd,jhd->hij", tq, tk.repeat_interleave(2, 1)) * 8 ** -0.5
    out = torch.einsum("hij,jhd->ihd", s.softmax(-1), tv.repeat_interleave(2, 1))
    torch.autograd.backward((out, s.logsumexp(-1).T), (torch.tensor(do), torch.tensor(dl)))
    for name, t in (("dq", tq), ("dk", tk), ("dv", tv)):
        assert np.allclose(r[name], t.grad.numpy())


def test_attention_grad_refusals():
    from hi3d_amd import attention

    q, k, v = _qkv()
    with pytest.raises(ValueError, match="ROCm GPU only"):
        attention.attend_grad(q, k, v, q, torch.zeros(4, 2), q)
    with pytest.raises(ValueError, match="ROCm GPU only"):
        attention.attend(q.requires_grad_(True), k, v)


def test_attention_grad_c_refusals():
    from hi3d_amd import _lib

    def call(out=4096, lse=4096, dout=4096, dlse=None, dq=4096, dk=4096, dv=4096, work=4096, size=1 << 30, **kw):
        _lib.call("hi3d_attention_backward", ctypes.byref(_desc(**kw)), out, lse, dout, dlse, dq, dk, dv, work, size, None)

    call(dq=None, dk=None, dv=None)
    call(total_q=0, len_q=0, total_k=0, len_k=0)
    for match, kw in [("together", dict(dk=None)), ("together", dict(dv=None)), ("null", dict(out=None)),
                      ("null", dict(lse=None)), ("null", dict(dout=None)), ("aligned", dict(dq=4100)),
                      ("aligned", dict(work=4104)), ("too small", dict(size=8)), ("too small", dict(work=None)),
                      ("type 0", dict(dtype=_lib.F32)), ("without a segment", dict(batch=0, cu_q=64, cu_k=64))]:
        with pytest.raises(ValueError, match=match):
            call(**kw)
    query = lambda **kw: _lib.query("hi3d_attention_backward_workspace", ctypes.byref(_desc(**kw)))  # noqa: E731
    assert query() > 0
    assert query(total_q=4096, len_q=4096) > 4096 * 4 * 4 + 2 * 4 * 2 * 64 * 4
    with pytest.raises(ValueError, match="null"):
        _lib.query("hi3d_attention_backward_workspace", None)


def test_token_attention_refusals():
    from hi3d_amd import torso

    for bad in ((100, 3), (96, 4, 3), (96, 0), (96, 24), (512, 2)):
        with pytest.raises(ValueError):
            torso.TokenAttention(*bad)
    block = torso.TokenAttention(64, 1)
    assert block.half().frequencies(torch.device("cpu")).dtype == torch.float64
    cache = torso.KeyValueCache(2, 4, 1, 64, device="cpu")
    cache.extend(0, torch.ones(3, 1, 64), torch.ones(3, 1, 64))
    with pytest.raises(ValueError, match="no room for 2"):
        cache.extend(0, torch.ones(2, 1, 64), torch.ones(2, 1, 64))
    cache.append(torch.full((2, 1, 64), 2.0), torch.zeros(2, 1, 64))
    assert cache.lens.tolist() == [4, 1] == cache.used and cache.k[0, 3, 0, 0] == 2 and cache.k[1, 0, 0, 0] == 2
    with pytest.raises(ValueError, match="sequence 0 holds 4 of 4"):
        cache.append(torch.ones(2, 1, 64), torch.ones(2, 1, 64))
    with pytest.raises(ValueError, match="one sequence"):
        block.float()(torch.zeros(2, 64), torch.zeros(2, 3, dtype=torch.int32), cache=cache)
