"""Attention and its gradients at sizes that small tests do not reach: 256 rows to a workgroup
(small heads, more than 2,048 such workgroups), streamed caches of several sequences. Bounds as
in the small tests."""

from __future__ import annotations

import pytest
import torch

from test_gpu_attention import _check_forward, _cu, _tensors
from test_gpu_attention_grad import _check, _grads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,masked,causal", [(32, False, False), (64, False, True), (64, True, False), (40, True, True)])
def test_wide_row_tiles(cuda, d, masked, causal):
    from hi3d_amd import attention

    lengths, keys = [33001, 1, 400, 33130], [150, 3, 170, 201]
    cu_q, cu_k = _cu(lengths), _cu(keys)
    q, k, v = _tensors(int(cu_q[-1]), int(cu_k[-1]), 8, 8, d, torch.bfloat16)
    mask = (torch.rand(int(cu_k[-1]), generator=torch.Generator().manual_seed(1)) < 0.7).cuda() if masked else None
    out, lse = attention.attend(q, k, v, attention.offsets(lengths), attention.offsets(keys), causal=causal,
                                key_mask=mask, return_lse=True)
    _check_forward(out, lse, q, k, v, cu_q, cu_k, causal=causal, mask=mask)


def test_gradients_of_many_rows(cuda):
    from hi3d_amd import attention

    lengths, keys = [9001, 1, 400, 9130], [150, 3, 170, 201]
    cu_q, cu_k = _cu(lengths), _cu(keys)
    q, k, v = _tensors(int(cu_q[-1]), int(cu_k[-1]), 8, 4, 64, torch.float16)
    dout = _tensors(int(cu_q[-1]), 1, 8, 1, 64, torch.float16, seed=3)[0]
    grads = _grads(q, k, v, dout, attention.offsets(lengths), attention.offsets(keys))
    _check(grads, q, k, v, dout, cu_q, cu_k)


def test_streamed_caches_of_several_sequences(cuda):
    """300 MB of keys and values, used to different lengths, against the same caches one by one
    (which are small enough to be held)."""
    from hi3d_amd import attention

    batch, room, hq, hk, d = 5, 30011, 8, 4, 128
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn((batch, room, hk, d), generator=g, device="cuda").half() for _ in range(2))
    q = torch.randn((batch, 1, hq, d), generator=g, device="cuda").half()
    lens = torch.tensor([30011, 17, 0, 29999, 12345], dtype=torch.int32, device="cuda")
    out = attention.attend(q, k, v, lens_k=lens)
    assert k.numel() * 4 > 256 << 20
    for b, n in enumerate(lens.tolist()):
        kk, vv = (x[b, :n].double().repeat_interleave(hq // hk, 1).transpose(0, 1) for x in (k, v))
        s = (kk * q[b, 0].double()[:, None]).sum(-1) * d ** -0.5
        p = torch.softmax(s, -1) if n else s
        want = (p[..., None] * vv).sum(1)
        size = (p[..., None] * vv.abs()).sum(1)
        # p and the output rounded to half a step each; fp32 sums of 30,000 terms in parts: 2^-14
        room_ = 2.0 ** -11 * (size + want.abs()) + 2.0 ** -14 * size + 2.0 ** -24
        assert bool(((out[b, 0].double() - want).abs() <= room_).all())
