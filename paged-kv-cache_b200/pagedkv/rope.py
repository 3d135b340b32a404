"""The angle table that B200Backend.rope_and_cache reads."""

from __future__ import annotations

import numpy as np


def rope_table(max_position: int, rotary_dim: int, base: float = 10000.0, inv_freq=None) -> np.ndarray:
    """f32 [max_position][rotary_dim]: for position p and pair j the cosine of
    p * inv_freq[j] in column j and its sine in column rotary_dim / 2 + j.
    inv_freq defaults to base ** (-2 j / rotary_dim); pass scaled frequencies
    for an extended context. The angles are taken in 64 bits: at position 10^5
    an f32 angle is already 4e-3 off. Build it once per model and keep it on
    the device."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and at least 2")
    if max_position < 1:
        raise ValueError("max_position must be positive")
    if inv_freq is None:
        inv_freq = float(base) ** (-np.arange(0, rotary_dim, 2, dtype=np.float64) / rotary_dim)
    inv_freq = np.asarray(inv_freq, dtype=np.float64)
    if inv_freq.shape != (rotary_dim // 2,):
        raise ValueError("inv_freq must hold rotary_dim / 2 frequencies")
    angle = np.arange(max_position, dtype=np.float64)[:, None] * inv_freq
    return np.concatenate([np.cos(angle), np.sin(angle)], axis=1).astype(np.float32)
