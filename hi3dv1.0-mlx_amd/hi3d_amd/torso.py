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
    None, or bool ``[batch, length]`` with False at the keys that a prompt's mask hid. ``shared``:
    None, or the cache of one sequence whose keys come before those of every sequence here (a common
    beginning, which is kept and read once)."""

    def __init__(self, batch: int, length: int, heads: int, dim: int, dtype: torch.dtype = torch.float16,
                 device: torch.device | str = "cuda", shared: KeyValueCache | None = None):
        self.k = torch.zeros((batch, length, heads, dim), dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.used = [0] * batch
        self.mask: torch.Tensor | None = None
        self._rows = torch.arange(batch, device=device)
        if shared is not None:
            if len(shared.used) != 1 or shared.shared is not None:
                raise ValueError("what sequences share is the cache of one sequence that shares nothing itself")
            if shared.k.shape[2:] != self.k.shape[2:] or shared.k.dtype != dtype or shared.k.device != self.k.device:
                raise ValueError(f"shared keys must be [.., {heads}, {dim}] of {dtype} on {self.k.device}")
        self.shared = shared

    def shared_keys(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
        """Keys, values and mask that the sequences share, as far as they are in use."""
        n = self.shared.used[0]
        return self.shared.k[0, :n], self.shared.v[0, :n], None if self.shared.mask is None else self.shared.mask[0, :n]

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
    values of a head turn (all by default) by ``axes`` positions a token. Scores may be capped
    (``cap``), fall with the distance of tokens in their order (``slopes``: :func:`attention.head_slopes`),
    and take a learned bias of that distance: ``buckets`` of them up to ``far`` tokens apart
    (:func:`attention.relative_buckets`), the parameter ``relative_bias [buckets, heads]``, zeros at first."""

    def __init__(self, channels: int, heads: int, key_heads: int | None = None, *, axes: int = 3, rot: int | None = None,
                 layout: str = "interleaved", base: float = 10000.0, causal: bool = False, bias: bool = True,
                 cap: float | None = None, slopes: bool = False, buckets: int = 0, far: int = 128,
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
        if cap is not None and not 1e-6 <= cap <= 1024.0:
            raise ValueError(f"a cap must be positive and at most 1024 (got {cap})")
        self._fixed: dict[torch.device, dict] = {torch.device("cpu"): {}}  # terms without a gradient: no buffers either
        if cap is not None:
            self._fixed[torch.device("cpu")]["cap"] = cap
        if slopes:
            self._fixed[torch.device("cpu")]["slopes"] = attention.head_slopes(heads, "cpu")
        self.relative_bias = None
        if buckets:
            self._fixed[torch.device("cpu")]["buckets"] = attention.relative_buckets(buckets, far, causal=causal, device="cpu")
            self.relative_bias = nn.Parameter(torch.zeros((buckets, heads), dtype=dtype, device=device))

    def frequencies(self, device: torch.device) -> torch.Tensor:
        """The float64 frequencies on ``device`` (no buffer: a module's cast would round them)."""
        if device not in self._freqs:
            with torch.inference_mode(False):  # kept past a first call in that mode, for gradients too
                self._freqs[device] = self._freqs[torch.device("cpu")].to(device)
        return self._freqs[device]

    def terms(self, device: torch.device) -> dict:
        """What :func:`attention.attend` takes for the scores' terms."""
        if device not in self._fixed:
            with torch.inference_mode(False):
                self._fixed[device] = {n: t.to(device) if torch.is_tensor(t) else t
                                       for n, t in self._fixed[torch.device("cpu")].items()}
        fixed = self._fixed[device]
        return fixed if self.relative_bias is None else dict(fixed, bias=self.relative_bias)

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
                key_mask: torch.Tensor | None = None, cache: KeyValueCache | None = None,
                prefix: torch.Tensor | None = None) -> torch.Tensor:
        """``x [N, C]`` with ``positions [N, axes]``, objects one after another at ``offsets``
        (:func:`attention.offsets`; one object without). ``cache``: takes the keys and values of
        the one sequence of a prompt, or of its next part, which also sees the keys that the
        cache holds or shares already (as constants, where gradients are wanted). ``key_mask``: of
        ``x``'s own tokens; a cache keeps it for what comes after. ``prefix`` (int32, one per object; of a
        causal block): so many first tokens are seen by all tokens of their object."""
        if cache is not None and (offsets is not None or len(cache.used) != 1):
            raise ValueError("a prompt fills the cache of one sequence")
        if prefix is not None and (not self.causal or cache is not None):
            raise ValueError("a prefix belongs to the objects of a causal block, without a cache")
        q, k, v = self.project(x, positions)
        terms = self.terms(x.device)
        if prefix is not None:
            terms = dict(terms, prefix=prefix)
        if cache is not None:
            self._check_type(cache, k)
            held = cache.used[0]
            recorded = torch.is_grad_enabled() and (k.requires_grad or self._learns_bias())
            cache.extend(0, k, v, key_mask)
            used = cache.used[0]
            shared = cache.shared is not None and cache.shared.used[0] > 0
            if shared and not recorded:
                mask = None if cache.mask is None else cache.mask[:, :used]
                pk, pv, pm = cache.shared_keys()
                y = attention.attend_shared(q[None], pk, pv, cache.k[:, :used], cache.v[:, :used], causal=self.causal,
                                            shared_mask=pm, key_mask=mask, **terms)
                return self.out(y.reshape(x.shape[0], self.heads * self.dim))
            if held and cache.mask is not None:
                key_mask = cache.mask[0, :used]
                key_mask = key_mask.clone() if recorded else key_mask
            if held and recorded:  # copies: autograd keeps them, and the cache changes with every token
                k, v = torch.cat([cache.k[0, :held], k]), torch.cat([cache.v[0, :held], v])
            elif held:
                k, v = cache.k[0, :used], cache.v[0, :used]
            if shared:
                pk, pv, pm = cache.shared_keys()
                k, v = torch.cat([pk, k]), torch.cat([pv, v])
                if pm is not None or key_mask is not None:
                    ones = [torch.ones(n, dtype=torch.bool, device=x.device) for n in (pk.shape[0], used)]
                    key_mask = torch.cat([ones[0] if pm is None else pm, ones[1] if key_mask is None else key_mask.bool()])
        y = attention.attend(q, k, v, offsets, causal=self.causal, key_mask=key_mask, **terms)
        return self.out(y.reshape(x.shape[0], self.heads * self.dim))

    def _learns_bias(self) -> bool:
        return self.relative_bias is not None and self.relative_bias.requires_grad

    @torch.no_grad()
    def step(self, x: torch.Tensor, positions: torch.Tensor, cache: KeyValueCache) -> torch.Tensor:
        """One new token ``x [batch, C]`` of every sequence of ``cache``, which takes its key and
        value; each sees all keys of its sequence, and of what the sequences share, that no mask hid."""
        q, k, v = self.project(x, positions)
        self._check_type(cache, k)
        cache.append(k, v)
        terms = self.terms(x.device)
        if cache.shared is not None:
            pk, pv, pm = cache.shared_keys()
            y = attention.attend_shared(q[:, None], pk, pv, cache.k, cache.v, lens_k=cache.lens, shared_mask=pm,
                                        key_mask=cache.mask, **terms)
        else:
            y = attention.attend(q[:, None], cache.k, cache.v, lens_k=cache.lens, key_mask=cache.mask, **terms)
        return self.out(y.reshape(x.shape[0], self.heads * self.dim))
