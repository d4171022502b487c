"""Matrices in 8 bits on the device, and the C ABI's calls on them and on gated
layers (ember_amd.capi).  GPU tests only."""

from __future__ import annotations

import numpy as np

import gpu_helpers as G
from ember_amd import capi
from ember_amd.capi import DeviceArray
from oracle import feedforward as ff
from serving_helpers import Bytes, U, ptr

ACT = dict(gelu=1, silu=2)


def arr(x):
    return None if x is None else DeviceArray.from_numpy(x)


class Rows8:
    """A matrix of the given size whose bytes are `fill`, or the given ones."""

    def __init__(self, rows, cols, fill=0xA5, codes=None, scales=None):
        self.rows, self.cols = rows, cols
        blank = lambda n: np.full((rows, n), fill, np.uint8)  # noqa: E731
        self.codes = Bytes(blank(ff.groups(cols) * 128) if codes is None else codes)
        self.scales = Bytes(blank(-(-ff.groups(cols) // 4) * 4) if scales is None else scales)
        self.view = capi.Rows8View(self.codes.ptr, self.scales.ptr, rows, cols)

    @classmethod
    def of(cls, x):
        """x rounded by the oracle."""
        codes, scales = ff.quantise8(x)
        return cls(*x.shape, codes=codes, scales=scales)

    def bytes(self):
        return self.codes.numpy(), self.scales.numpy()

    def values(self):
        return ff.values8(*self.bytes(), self.cols)


def check_held(m, exact, off):
    """m holds what rounding numbers within `off` of `exact` (float64) gives: a
    scale that fits the largest of each group, and elements at most half a step
    away (2^-4 of a number, 2^-10 of the scale for the smallest codes)."""
    codes, scales = m.bytes()
    rows, cols = exact.shape
    n = ff.groups(cols)
    pad = lambda x: np.pad(x, ((0, 0), (0, n * 128 - cols))).reshape(rows, n, 128)  # noqa: E731
    least = lambda a: np.maximum(np.ceil(np.log2(np.where(a > 0, a, 2.0 ** -150) / 448)), -119) + 127  # noqa: E731
    low, high = ((np.abs(pad(exact)) + s * pad(off)).max(-1) for s in (-1, 1))
    fits = (scales[:, :n] >= least(low)) & (scales[:, :n] <= least(high))
    assert (fits | ((low <= 0) & (scales[:, :n] == 127))).all()  # a group that may be zeros may have their byte
    assert (scales[:, n:] == 127).all() and (codes[:, cols:] == 0).all()
    step = np.repeat(2.0 ** (scales.astype(np.float64) - 127), 128, 1)[:, :cols]
    tol = off + 2.0 ** -4 * (np.abs(exact) + off) + 2.0 ** -10 * step
    got = m.values()
    assert np.isfinite(got).all()
    bad = ~(np.abs(got - exact) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size}"


def linear8(a, w, bias=None, residual=None, act=0, log=None):
    G.say(f"linear8_fwd n={a.rows} m={w.rows} k={a.cols} bias={bias is not None} residual={residual is not None} act={act}")
    out = DeviceArray.from_numpy(np.full((a.rows, w.rows), G.SENTINEL, np.float32))
    b, r = arr(bias), arr(residual)
    capi.launch_log_reset()
    rc = capi.lib().linear8_fwd(a.view, w.view, ptr(b), ptr(r), out.ptr, act)
    if log is not None:
        log.extend(capi.launch_log())
    capi.check(rc, "linear8_fwd")
    return out.numpy()


def gated8(a, w, bias, act, log=None):
    G.say(f"gated8_fwd n={a.rows} hidden={w.rows // 2} k={a.cols} bias={bias is not None} act={act}")
    h, b = Rows8(a.rows, w.rows // 2), arr(bias)
    capi.launch_log_reset()
    rc = capi.lib().gated8_fwd(a.view, w.view, ptr(b), h.view, ACT[act])
    if log is not None:
        log.extend(capi.launch_log())
    capi.check(rc, "gated8_fwd")
    return h


def product(a, w):
    """a w^T of two Rows8 in float64, and the sums of the products' sizes."""
    x, y = a.values(), w.values()
    return x @ y.T, np.abs(x) @ np.abs(y).T


def sum_error(reach, k):
    """How far an fp32 sum of k exact products may be off: a step of the largest
    partial sum for each (the matrix cores cut off what they shift out)."""
    return 2 * U * (k + 4) * reach


def gate_error(act, pre, off):
    """How far act(gate) * up may be off where both sums are off by `off`: the slope
    of either activation is below 1.2, and its value is formed to 8 half steps of
    |gate| (1 + tanh cancels far below 0)."""
    half = pre.shape[-1] // 2
    gate, up, og, ou = pre[:, :half], pre[:, half:], off[:, :half], off[:, half:]
    value = np.abs(ff.activate(act, gate)[0])
    wrong = 1.2 * og + 8 * U * np.abs(gate)
    return wrong * (np.abs(up) + ou) + value * (ou + 4 * U * np.abs(up))
