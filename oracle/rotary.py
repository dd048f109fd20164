"""Rotary positions restated in numpy, in 64 bits: each pair of dims as a complex
number, multiplied by scale * exp(i p f).

No counterpart in the reference, which has no positions.
"""
from __future__ import annotations

import numpy as np


def rotate(x, positions, freqs, interleaved=False, scale=1.0, back=False):
    """x [..., N, D] (float64) at positions [..., N] or [N]; freqs [R / 2]."""
    R = 2 * len(freqs)
    y = np.array(x, np.float64)
    r = y[..., :R]
    x1, x2 = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :R // 2], r[..., R // 2:])
    angle = np.asarray(positions, np.float64)[..., None] * np.asarray(freqs, np.float64)
    with np.errstate(invalid="ignore"):
        z = (x1 + 1j * x2) * (scale * np.exp((-1j if back else 1j) * angle))
    if interleaved:
        r[..., 0::2], r[..., 1::2] = z.real, z.imag
    else:
        r[..., :R // 2], r[..., R // 2:] = z.real, z.imag
    return y


def pair_size(x, freqs, interleaved=False):
    """|x1| + |x2| of each value's pair (|x| itself past R): what errors of the factors are multiplied by."""
    R = 2 * len(freqs)
    a = np.abs(np.array(x, np.float64))
    if interleaved:
        s = a[..., 0:R:2] + a[..., 1:R:2]
        a[..., 0:R:2], a[..., 1:R:2] = s, s
    else:
        s = a[..., :R // 2] + a[..., R // 2:R]
        a[..., :R // 2], a[..., R // 2:R] = s, s
    return a
