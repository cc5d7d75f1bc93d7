"""Rotary positions and head norms in float64 numpy, with the magnitudes of the terms."""
import numpy as np


def angles(positions, inv_freq):
    a = np.asarray(positions, np.float64)[..., None, None] * np.asarray(inv_freq, np.float64)
    return np.cos(a), np.sin(a)


def turn(x, positions, inv_freq, layout, scale, sign=1.0):
    """(s R(sign p f) x, sum of the terms' magnitudes) of x [B, L, H, D], positions [B, L]."""
    x = np.asarray(x, np.float64)
    n = 2 * len(inv_freq)
    c, s = angles(positions, inv_freq)
    c, s = c * scale, sign * s * scale
    ia, ib = (np.arange(n // 2), np.arange(n // 2) + n // 2) if layout == "half" else (np.arange(0, n, 2), np.arange(1, n, 2))
    a, b = x[..., ia], x[..., ib]
    y, m = x.copy(), np.abs(x)
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    m[..., ia], m[..., ib] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
    return y, m


def norm(x, w, eps):
    """(x r, r) with r = (mean x^2 + eps)^-1/2; times w outside."""
    x = np.asarray(x, np.float64)
    r = (np.mean(x * x, -1, keepdims=True) + eps) ** -0.5
    return x * r, r


def norm_turn(x, w, positions, inv_freq, layout, scale, eps):
    xr, _ = norm(x, w, eps)
    return turn(xr * np.asarray(w, np.float64), positions, inv_freq, layout, scale)


def norm_turn_grads(x, w, g, positions, inv_freq, layout, scale, eps):
    """((dx, magnitude), (dw, magnitude))."""
    xr, r = norm(x, w, eps)
    w = np.asarray(w, np.float64)
    dy, my = turn(g, positions, inv_freq, layout, scale, -1.0)
    t = dy * w
    m = np.mean(t * xr, -1, keepdims=True)
    mm = np.mean(my * np.abs(w * xr), -1, keepdims=True)
    return ((r * (t - xr * m), r * (my * np.abs(w) + np.abs(xr) * mm)),
            ((dy * xr).sum((0, 1, 2)), (my * np.abs(xr)).sum((0, 1, 2))))
