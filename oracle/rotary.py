"""Rotary positions in float64 (the torso's rotation of queries and keys by voxel
coordinates, src/sparc3d/nn/rope.py)."""

from __future__ import annotations

import numpy as np


def rotate(x, positions, freqs, layout="half", scale=1.0, inverse=False) -> np.ndarray:
    """``x [N, H, D]``, ``positions [N, axes]``, ``freqs [axes, rot / 2]``."""
    x = np.asarray(x, np.float64)
    turn = np.exp((-1j if inverse else 1j) * (np.asarray(positions, np.float64) @ np.asarray(freqs, np.float64)))[:, None]
    rot = 2 * freqs.shape[1]
    at = np.arange(rot).reshape(2, -1) if layout == "half" else np.arange(rot).reshape(-1, 2).T
    z = (x[..., at[0]] + 1j * x[..., at[1]]) * turn * scale
    y = x.copy()
    y[..., at[0]], y[..., at[1]] = z.real, z.imag
    return y
