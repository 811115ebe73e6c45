"""Self attention of a torso block on the token operators: projection, rotary positions,
attention within each object and the output projection, trainable; and the same block
stepping one token at a time over a cache. The refiner's attention modules
(src/sparc3d/nn/sparse/attention/modules.py, src/sparc3d/nn/rope.py) have this order of
steps and a root mean square norm of queries and keys besides, which is not formed here:
this is not a drop-in for them, and the refiner itself keeps no cache."""

from __future__ import annotations

import torch
from torch import nn

from . import attention, rotary


class KeyValueCache:
    """Room for ``length`` keys and values of each of ``batch`` sequences, ``[batch, length,
    heads, dim]``, and how many are in use: ``lens`` on the GPU, ``used`` on the host. ``mask``:
    None, or bool ``[batch, length]`` with False at the keys that a prompt's mask hid."""

    def __init__(self, batch: int, length: int, heads: int, dim: int, dtype: torch.dtype = torch.float16,
                 device: torch.device | str = "cuda"):
        self.k = torch.zeros((batch, length, heads, dim), dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.used = [0] * batch
        self.mask: torch.Tensor | None = None
        self._rows = torch.arange(batch, device=device)

    def _check(self, count: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """What is refused is refused before anything is written."""
        shape = (count, *self.k.shape[2:])
        for name, x in (("k", k), ("v", v)):
            if x.shape != shape or x.device != self.k.device:
                raise ValueError(f"{name} must be {list(shape)} on {self.k.device} (got {list(x.shape)} on {x.device})")

    def _room(self, which: int, count: int) -> None:
        if not 0 <= which < len(self.used):
            raise ValueError(f"no sequence {which} of {len(self.used)}")
        if self.used[which] + count > self.k.shape[1]:
            raise ValueError(f"sequence {which} holds {self.used[which]} of {self.k.shape[1]} keys: no room for {count}")

    def extend(self, which: int, k: torch.Tensor, v: torch.Tensor, key_mask: torch.Tensor | None = None) -> None:
        """Adds the keys and values ``[n, heads, dim]`` of a prompt to one sequence; those where
        ``key_mask [n]`` is False are there, but not seen."""
        n = int(k.shape[0])
        self._room(which, n)
        self._check(n, k, v)
        at = self.used[which]
        if key_mask is not None:
            if key_mask.dtype not in (torch.bool, torch.uint8) or key_mask.shape != (n,) or key_mask.device != k.device:
                raise ValueError(f"key_mask must be bool [{n}] on {k.device}")
            if self.mask is None:
                self.mask = torch.ones(self.k.shape[:2], dtype=torch.bool, device=self.k.device)
            self.mask[which, at:at + n] = key_mask
        elif self.mask is not None:
            self.mask[which, at:at + n] = True
        self.k[which, at:at + n] = k.detach()
        self.v[which, at:at + n] = v.detach()
        self.used[which] += n
        self.lens[which] = self.used[which]

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """Adds one key and value ``[batch, heads, dim]`` to every sequence."""
        self._check(len(self.used), k, v)
        for b in range(len(self.used)):
            self._room(b, 1)
        at = self.lens.long()
        self.k[self._rows, at] = k.detach().to(self.k.dtype)
        self.v[self._rows, at] = v.detach().to(self.v.dtype)
        if self.mask is not None:
            self.mask[self._rows, at] = True
        self.lens += 1
        self.used = [n + 1 for n in self.used]


class TokenAttention(nn.Module):
    """``x + ...`` is the caller's: this is ``out(attend(rotate(qkv(x))))`` of tokens ``[N, C]``.

    ``key_heads`` fewer than ``heads`` share keys and values between query heads; ``rot``
    values of a head turn (all by default) by ``axes`` positions a token."""

    def __init__(self, channels: int, heads: int, key_heads: int | None = None, *, axes: int = 3, rot: int | None = None,
                 layout: str = "interleaved", base: float = 10000.0, causal: bool = False, bias: bool = True,
                 dtype: torch.dtype = torch.float16, device: torch.device | str | None = None):
        super().__init__()
        key_heads = heads if key_heads is None else key_heads
        if heads < 1 or key_heads < 1 or channels % heads or heads % key_heads:
            raise ValueError(f"{channels} channels, {heads} heads and {key_heads} key heads do not divide")
        self.heads, self.key_heads, self.dim, self.causal, self.layout = heads, key_heads, channels // heads, causal, layout
        if self.dim % 8 or self.dim > 128:
            raise ValueError(f"head size must be a multiple of 8 up to 128 (got {self.dim})")
        self.qkv = nn.Linear(channels, (heads + 2 * key_heads) * self.dim, bias=bias, dtype=dtype, device=device)
        self.out = nn.Linear(channels, channels, bias=bias, dtype=dtype, device=device)
        self._freqs = {torch.device("cpu"): rotary.frequencies(self.dim if rot is None else rot, axes=axes, base=base)}

    def frequencies(self, device: torch.device) -> torch.Tensor:
        """The float64 frequencies on ``device`` (no buffer: a module's cast would round them)."""
        if device not in self._freqs:
            self._freqs[device] = self._freqs[torch.device("cpu")].to(device)
        return self._freqs[device]

    def project(self, x: torch.Tensor, positions: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Turned queries and keys, and values, of tokens ``x [N, C]``."""
        heads = self.qkv(x).view(x.shape[0], self.heads + 2 * self.key_heads, self.dim)
        q, k, v = heads.split([self.heads, self.key_heads, self.key_heads], 1)
        q, k = rotary.rotate_qk(q, k, positions, self.frequencies(x.device), layout=self.layout)
        return q, k, v

    @staticmethod
    def _check_type(cache: KeyValueCache, k: torch.Tensor) -> None:
        if cache.k.dtype != k.dtype:
            raise ValueError(f"the cache must be of the block's {k.dtype} (got {cache.k.dtype})")

    def forward(self, x: torch.Tensor, positions: torch.Tensor, offsets: torch.Tensor | None = None, *,
                key_mask: torch.Tensor | None = None, cache: KeyValueCache | None = None) -> torch.Tensor:
        """``x [N, C]`` with ``positions [N, axes]``, objects one after another at ``offsets``
        (:func:`attention.offsets`; one object without). ``cache``: takes the keys and values of
        the one sequence of a prompt, or of its next part, which also sees the keys that the
        cache holds already (as constants, where gradients are wanted). ``key_mask``: of ``x``'s own
        tokens; a cache keeps it for what comes after."""
        if cache is not None and (offsets is not None or len(cache.used) != 1):
            raise ValueError("a prompt fills the cache of one sequence")
        q, k, v = self.project(x, positions)
        if cache is not None:
            self._check_type(cache, k)
            held, recorded = cache.used[0], torch.is_grad_enabled() and k.requires_grad
            cache.extend(0, k, v, key_mask)
            if held and cache.mask is not None:
                key_mask = cache.mask[0, :cache.used[0]]
                key_mask = key_mask.clone() if recorded else key_mask
            if held and recorded:  # copies: autograd keeps them, and the cache changes with every token
                k, v = torch.cat([cache.k[0, :held], k]), torch.cat([cache.v[0, :held], v])
            elif held:
                k, v = cache.k[0, :cache.used[0]], cache.v[0, :cache.used[0]]
        y = attention.attend(q, k, v, offsets, causal=self.causal, key_mask=key_mask)
        return self.out(y.reshape(x.shape[0], self.heads * self.dim))

    @torch.no_grad()
    def step(self, x: torch.Tensor, positions: torch.Tensor, cache: KeyValueCache) -> torch.Tensor:
        """One new token ``x [batch, C]`` of every sequence of ``cache``, which takes its key and
        value; each sees all keys of its sequence that no mask hid."""
        q, k, v = self.project(x, positions)
        self._check_type(cache, k)
        cache.append(k, v)
        y = attention.attend(q[:, None], cache.k, cache.v, lens_k=cache.lens, key_mask=cache.mask)
        return self.out(y.reshape(x.shape[0], self.heads * self.dim))
