"""Head norms and position rotation in float64 numpy, from the formulas.

    n = x * r,  r = (mean x^2 + eps)^-1/2,  y = R(pos) (n * w)
    g = R(pos)^T dy,  dx = r (w g - n mean(w g n)),  dw = sum g n
"""

from __future__ import annotations

import numpy as np


def rotation(x, cos, sin, interleaved=False):
    """x [token, head, dim]; cos, sin [token, rot / 2] of each token's position."""
    x = np.asarray(x, dtype=np.float64)
    y = x.copy()
    half = cos.shape[1]
    rot = 2 * half
    first = np.arange(half) * 2 if interleaved else np.arange(half)
    second = first + 1 if interleaved else first + half
    c, s = cos[:, None].astype(np.float64), sin[:, None].astype(np.float64)
    a, b = x[..., :rot][..., first], x[..., :rot][..., second]
    y[..., first] = a * c - b * s
    y[..., second] = b * c + a * s
    return y


def norm_rope(x, weight, cos, sin, eps=1e-6, interleaved=False):
    x = np.asarray(x, dtype=np.float64)
    if weight is not None:
        r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        x = x * r * np.asarray(weight, dtype=np.float64)
    return rotation(x, cos, sin, interleaved)


def norm_rope_grad(x, weight, dy, cos, sin, eps=1e-6, interleaved=False):
    """(dx, dw); dw is None without a weight."""
    x, dy = np.asarray(x, dtype=np.float64), np.asarray(dy, dtype=np.float64)
    g = rotation(dy, cos, -np.asarray(sin), interleaved)
    if weight is None:
        return g, None
    w = np.asarray(weight, dtype=np.float64)
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n = x * r
    wg = w * g
    return r * (wg - n * (wg * n).mean(-1, keepdims=True)), (g * n).sum((0, 1))
