"""Plain NumPy forms, in 64 bits, of RMS norm, matrices in 8 bits and gated
feed-forward layers.  Written from the formulas; loops where they are clearest."""

from __future__ import annotations

import numpy as np

GROUP = 128


def _e4m3():
    """The 127 sizes of E4M3, by code."""
    n = np.arange(127)
    e, f = n >> 3, n & 7
    return np.where(e > 0, (1 + f / 8) * 2.0 ** (e - 7.0), f * 2.0 ** -9)


E4M3 = _e4m3()


def groups(cols):
    return -(-cols // GROUP)


def quantise8(x):
    """Codes (rows, groups * 128) and scale bytes (rows, groups in whole fours) of
    float32 x (rows, cols)."""
    x = np.asarray(x, np.float32)
    rows, cols = x.shape
    g = np.zeros((rows, groups(cols) * GROUP))
    g[:, :cols] = x
    g = g.reshape(rows, -1, GROUP)
    amax = np.abs(g).max(-1)
    held = amax < 2.0 ** 127  # false for NaN
    safe = np.where(held & (amax > 0), amax, 448.0)
    e = np.maximum(np.ceil(np.log2(safe / 448)), -119)
    byte = np.where(held, np.where(amax > 0, e + 127, 127), 255).astype(np.uint8)
    y = np.abs(np.where(held[..., None], g, 0)) * 2.0 ** -e[..., None]
    above = np.searchsorted(E4M3, y).clip(1, 126)  # E4M3[above - 1] < y <= E4M3[above], at the ends the nearest pair
    lo, hi = y - E4M3[above - 1], E4M3[above] - y
    code = np.where((hi < lo) | ((hi == lo) & (above % 2 == 0)), above, above - 1)
    code = np.where(held[..., None], code | (np.signbit(g) * 128), 0).astype(np.uint8)
    scales = np.full((rows, -(-groups(cols) // 4) * 4), 127, np.uint8)
    scales[:, :groups(cols)] = byte
    return code.reshape(rows, -1), scales


def values8(codes, scales, cols):
    """float64 (rows, cols) that codes and scale bytes stand for."""
    n = codes & 127
    size = np.where(n == 127, np.nan, E4M3[np.minimum(n, 126)]) * np.where(codes & 128, -1.0, 1.0)
    scale = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (size * np.repeat(scale, GROUP, -1)[:, :codes.shape[1]])[:, :cols]


def rmsnorm_fwd(s, gamma, eps):
    """y and rstd of the sums s (rows, d)."""
    s = np.asarray(s, np.float64)
    rstd = 1 / np.sqrt((s * s).mean(-1) + float(np.float32(eps)))
    return s * rstd[:, None] * np.asarray(gamma, np.float64), rstd


def rmsnorm_bwd(s, gamma, rstd, dy, dres=None):
    """dx and dgamma."""
    s, dy, rstd = np.asarray(s, np.float64), np.asarray(dy, np.float64), np.asarray(rstd, np.float64)[:, None]
    xhat, g = s * rstd, dy * np.asarray(gamma, np.float64)
    dx = rstd * (g - xhat * (g * xhat).mean(-1, keepdims=True))
    return dx if dres is None else dx + dres, (dy * xhat).sum(0)


def activate(act, x):
    """Value and slope of act "gelu" (0.5x(1 + tanh(0.8x))) or "silu"."""
    x = np.asarray(x, np.float64)
    if act == "gelu":
        t = np.tanh(0.8 * x)
        return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.4 * x * (1 - t * t)
    s = np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))
    return x * s, s + x * s * (1 - s)


def gate(act, pre):
    """h of both sums side by side (n, 2 hidden)."""
    half = pre.shape[-1] // 2
    return activate(act, pre[..., :half])[0] * pre[..., half:]


def gate_bwd(act, dh, pre):
    """The gradient of both sums."""
    half = pre.shape[-1] // 2
    value, slope = activate(act, pre[..., :half])
    return np.concatenate((dh * pre[..., half:] * slope, dh * value), -1)
