"""The definition of rotary positions and of the per-head norm in extended
precision (80-bit long double), for the tests of the attention layer's
operators."""
from __future__ import annotations

import numpy as np

LD = np.longdouble


def frequencies(n: int, base: float = 10000.0) -> np.ndarray:
    return base ** (-np.arange(n, dtype=np.float64) / n)


def angles(pos: np.ndarray, freqs: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """cos and sin [B, T, 1, R/2] of the f64 products position * frequency."""
    a = (pos.astype(np.float64)[..., None] * freqs).astype(LD)[:, :, None]
    return np.cos(a), np.sin(a)


def pairs(x: np.ndarray, R: int, layout: str):
    if layout == "half":
        return x[..., : R // 2], x[..., R // 2 : R]
    return x[..., 0:R:2], x[..., 1:R:2]


def join(x: np.ndarray, a: np.ndarray, b: np.ndarray, layout: str) -> np.ndarray:
    R = 2 * a.shape[-1]
    y = x.astype(LD).copy()
    if layout == "half":
        y[..., : R // 2], y[..., R // 2 : R] = a, b
    else:
        y[..., 0:R:2], y[..., 1:R:2] = a, b
    return y


def rotate(x, pos, freqs, layout, m=1.0, inverse=False):
    c, s = angles(pos, freqs)
    if inverse:
        s = -s
    a, b = pairs(x.astype(LD), 2 * len(freqs), layout)
    return join(x, LD(m) * (a * c - b * s), LD(m) * (b * c + a * s), layout)


def reach(x, freqs, layout, m=1.0):
    """|a| + |b| of every element's pair times the magnitude (|x| where no pair is): what a rounding of the
    rotation is relative to."""
    x = np.abs(x.astype(LD))
    a, b = pairs(x, 2 * len(freqs), layout)
    return join(x, LD(m) * (a + b), LD(m) * (a + b), layout)


def norm(x, eps):
    x = x.astype(LD)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + LD(eps))
    return x * r, r


def norm_rotate(x, gamma, eps, pos, freqs, layout, m=1.0):
    n, _ = norm(x, eps)
    return rotate(n * gamma.astype(LD), pos, freqs, layout, m)


def norm_rotate_backward(dy, x, gamma, eps, pos, freqs, layout, m=1.0):
    n, r = norm(x, eps)
    g = rotate(dy, pos, freqs, layout, m, inverse=True)
    dn = g * gamma.astype(LD)
    dx = r * (dn - n * (dn * n).mean(-1, keepdims=True))
    return dx, (g * n).sum((0, 1, 2))


def norm_backward_reach(dy, x, gamma, eps, freqs, layout, m=1.0):
    n, r = norm(x, eps)
    g = reach(dy, freqs, layout, m)
    dn = g * np.abs(gamma.astype(LD))
    n = np.abs(n)
    return r * (dn + n * (dn * n).mean(-1, keepdims=True)), (g * n).sum((0, 1, 2))
