"""RMS norm, 8-bit matrices and gated layers with more than 2^32 elements, rows past
a launch's, and the longest rows: some rows of each against float64."""

import ctypes

import numpy as np
import pytest

import gpu_helpers as G
from ember_amd import capi
from ember_amd.capi import DeviceArray
from feedforward_helpers import Rows8, U, arr, ff, gate_error, linear8, sum_error

pytestmark = pytest.mark.gpu

N, M, K = (1 << 20) + 37, 4100, 128
ROWS = [0, 1, 511, (1 << 20) - 1, 1 << 20, N - 2, N - 1]


def some(ptr, rows, row_bytes):
    """The bytes of some rows of a matrix on the device."""
    out = np.empty((len(rows), row_bytes), np.uint8)
    capi.lib().sync_device()
    for i, r in enumerate(rows):
        capi.lib().copy_from_device(out[i].ctypes.data, ctypes.c_void_p(ptr + r * row_bytes), row_bytes)
    capi.check(what="copy_from_device")
    return out


def floats(ptr, rows, cols):
    return some(ptr, rows, 4 * cols).view(np.float32)


class Blank8:
    """A Rows8 on the device alone."""

    def __init__(self, rows, cols):
        self.pitch, self.scale_pitch, self.cols = ff.groups(cols) * 128, -(-ff.groups(cols) // 4) * 4, cols
        self.codes, self.scales = DeviceArray((rows * self.pitch // 4,)), DeviceArray((-(-rows * self.scale_pitch // 4),))
        self.view = capi.Rows8View(self.codes.ptr, self.scales.ptr, rows, cols)

    def bytes(self, rows):
        return some(self.codes.ptr, rows, self.pitch), some(self.scales.ptr, rows, self.scale_pitch)


@pytest.fixture(scope="module")
def matrices():
    rng = np.random.default_rng(1)
    # Codes of 0.25 to 1.875 of either sign.
    codes = lambda n: (rng.integers(40, 64, (n, K)) + 128 * rng.integers(0, 2, (n, K))).astype(np.uint8)  # noqa: E731
    scales = lambda n: rng.integers(124, 128, (n, 4)).astype(np.uint8)  # noqa: E731
    return Rows8(N, K, codes=codes(N), scales=scales(N)), Rows8(2 * M, K, codes=codes(2 * M), scales=scales(2 * M))


def of_rows(m, rows):
    codes, scales = m.bytes()
    return ff.values8(codes[rows], scales[rows], m.cols)


def test_products_norms_and_rounding(matrices):
    a, both = matrices
    L = capi.lib()
    w = capi.Rows8View(both.codes.ptr, both.scales.ptr, M, K)
    x, gamma, rstd = DeviceArray((N, M)), arr(np.linspace(0.5, 1.5, M)), DeviceArray((N,))
    G.say("linear8_fwd, 2^32 elements")
    capi.check(L.linear8_fwd(a.view, w, None, None, x.ptr, 0), "linear8_fwd")
    av, wv = of_rows(a, ROWS), of_rows(both, slice(0, M))
    got = floats(x.ptr, ROWS, M)
    assert (np.abs(got - av @ wv.T) <= sum_error(np.abs(av) @ np.abs(wv).T, K)).all()
    # Rounded, and read back in place of what was rounded.
    m = Blank8(N, M)
    G.say("rows8_write, rows8_read, 2^32 elements")
    capi.check(L.rows8_write(m.view, x.ptr, M, 0), "rows8_write")
    codes, scales = ff.quantise8(got)
    for have, want in zip(m.bytes(ROWS), (codes, scales)):
        np.testing.assert_array_equal(have, want)
    capi.check(L.rows8_read(m.view, x.ptr, M), "rows8_read")
    held = ff.values8(codes, scales, M).astype(np.float32)
    np.testing.assert_array_equal(floats(x.ptr, ROWS, M), held)
    G.say("rmsnorm_fwd8, 2^32 elements")
    capi.check(L.rmsnorm_fwd8(x.ptr, None, gamma.ptr, None, m.view, 1e-5), "rmsnorm_fwd8")
    y, r = ff.rmsnorm_fwd(held, gamma.numpy(), 1e-5)
    G.say("rmsnorm_fwd, rmsnorm_bwd, 2^32 elements")
    out = DeviceArray((N, M))
    capi.check(L.rmsnorm_fwd(x.ptr, None, gamma.ptr, None, out.ptr, rstd.ptr, N, M, 1e-5), "rmsnorm_fwd")
    got = floats(out.ptr, ROWS, M)
    assert (np.abs(got - y) <= U * (1 + 2.0 ** -20) * np.abs(y)).all()
    for have, want in zip(m.bytes(ROWS), ff.quantise8(got)):
        np.testing.assert_array_equal(have, want)
    dgamma = DeviceArray((M,))
    m = None
    dx = DeviceArray((N, M))
    capi.check(L.rmsnorm_bwd(x.ptr, gamma.ptr, rstd.ptr, out.ptr, None, dx.ptr, dgamma.ptr, N, M), "rmsnorm_bwd")
    want, _ = ff.rmsnorm_bwd(held, gamma.numpy(), r, got.astype(np.float64))
    # The mean over a row: 8 terms to a lane, 6 steps over a wave, 16 waves, three roundings before: 45 half steps of what it adds up.
    g, xhat = got.astype(np.float64) * gamma.numpy(), held * r.reshape(-1, 1)
    mean = np.abs(g * xhat).mean(1, keepdims=True)
    assert (np.abs(floats(dx.ptr, ROWS, M) - want) <= U * r.reshape(-1, 1) * (6 * np.abs(g) + 55 * np.abs(xhat) * mean) + 2 * U * np.abs(want)).all()
    # dy = xhat * gamma, so dgamma / gamma is the columns' sum of xhat^2, over all columns
    # rows * d (1 - eps rstd^2): runs of 4097 rows summed in fp32 one by one, 4097 U of it.
    assert abs((dgamma.numpy().astype(np.float64) / gamma.numpy()).sum() / N / M - 1) <= 4200 * U + 1e-5 * float((r * r).max())


def test_transposed(matrices):
    """The last rows of what is written transposed from 2^32 elements."""
    a, both = matrices
    L = capi.lib()
    w = capi.Rows8View(both.codes.ptr, both.scales.ptr, M, K)
    x, m = DeviceArray((N, M)), Blank8(M, N)
    capi.check(L.linear8_fwd(a.view, w, None, None, x.ptr, 0), "linear8_fwd")
    G.say("rows8_write, transposed, 2^32 elements")
    capi.check(L.rows8_write(m.view, x.ptr, M, 1), "rows8_write")
    tail = list(range(N // 128 * 128, N))
    codes, scales = ff.quantise8(np.ascontiguousarray(floats(x.ptr, tail, M).T))
    rows = [0, 1, 2047, M - 1]
    have, byte = m.bytes(rows)
    np.testing.assert_array_equal(have[:, N // 128 * 128:], codes[rows])
    np.testing.assert_array_equal(byte[:, N // 128], scales[rows, 0])


def test_gated_layer_in_8_bits(matrices):
    a, w = matrices
    h = Blank8(N, M)
    G.say("gated8_fwd, 2^32 elements")
    capi.check(capi.lib().gated8_fwd(a.view, w.view, None, h.view, 2), "gated8_fwd")
    av, wv = of_rows(a, ROWS), of_rows(w, slice(0, 2 * M))
    pre, reach = av @ wv.T, np.abs(av) @ np.abs(wv).T
    exact = ff.gate("silu", pre)
    codes, scales = h.bytes(ROWS)
    step = np.repeat(2.0 ** (scales.astype(np.float64) - 127), 128, 1)[:, :M]
    off = gate_error("silu", pre, sum_error(reach, K))
    assert (np.abs(ff.values8(codes, scales, M) - exact) <= off + 2.0 ** -4 * (np.abs(exact) + off) + 2.0 ** -10 * step).all()


def test_gated_layer_in_fp32():
    n, hidden, d = (1 << 19) + 5, M, 4
    rng = np.random.default_rng(2)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    x, w, w_down, dy = f(n, d), f(d, 2 * hidden), f(hidden, d), f(n, d)
    dev = [arr(v) for v in (x, w, w_down, dy)]
    h, pre, dpre = DeviceArray((n, hidden)), DeviceArray((n, 2 * hidden)), DeviceArray((n, 2 * hidden))
    G.say("gated_fwd, gated_bwd, 2^32 elements")
    capi.check(capi.lib().gated_fwd(dev[0].ptr, dev[1].ptr, None, h.ptr, pre.ptr, n, hidden, d, 2), "gated_fwd")
    capi.check(capi.lib().gated_bwd(dev[3].ptr, dev[2].ptr, pre.ptr, dpre.ptr, n, hidden, d, 2), "gated_bwd")
    rows = [0, 1, 255, 256, 1 << 18, n - 6, n - 1]
    exact = x[rows].astype(np.float64) @ w
    got = floats(pre.ptr, rows, 2 * hidden).astype(np.float64)
    assert (np.abs(got - exact) <= 8 * U * (np.abs(x[rows]).astype(np.float64) @ np.abs(w))).all()
    kept = ff.gate("silu", got)
    assert (np.abs(floats(h.ptr, rows, hidden) - kept) <= gate_error("silu", got, 0 * got) + 2.0 ** -148).all()
    dh, reach = dy[rows].astype(np.float64) @ w_down.T, np.abs(dy[rows]).astype(np.float64) @ np.abs(w_down).T
    gate, up = got[:, :hidden], got[:, hidden:]
    # Terms: dh off by 8 U of its reach, slope and value by 8 U (1 + |gate|).
    slope = (1 + np.abs(gate)) * (1.2 + 8 * U)
    tol = 16 * U * np.concatenate((slope * np.abs(up) * reach, slope * reach), 1)
    assert (np.abs(floats(dpre.ptr, rows, 2 * hidden) - ff.gate_bwd("silu", dh, got)) <= tol + 2.0 ** -148).all()


def test_a_wide_gated_layer():
    """Halves of a row that lie more than 2^30 bytes apart."""
    hidden = (1 << 28) + 100
    w = np.tile(np.random.default_rng(3).standard_normal(1 << 20).astype(np.float32), 513)[:2 * hidden]
    x = np.float32([[0.5], [-2]])
    dx, dw, h, pre = arr(x), arr(w), DeviceArray((2, hidden)), DeviceArray((2, 2 * hidden))
    G.say(f"gated_fwd hidden={hidden}")
    capi.check(capi.lib().gated_fwd(dx.ptr, dw.ptr, None, h.ptr, pre.ptr, 2, hidden, 1, 2), "gated_fwd")
    for at in (0, (1 << 27) - 50, hidden - 100):
        cols = np.arange(at, at + 100)
        for r in (0, 1):
            both = np.concatenate((w[cols], w[hidden + cols])).astype(np.float64)[None] * x[r, 0]
            got = np.empty(100, np.float32)
            capi.lib().copy_from_device(got.ctypes.data, ctypes.c_void_p(h.ptr + 4 * (r * hidden + at)), 400)
            assert (np.abs(got - ff.gate("silu", both)[0]) <= gate_error("silu", both, 2 * U * np.abs(both))[0]).all()
    capi.check(what="copy_from_device")


@pytest.mark.parametrize("n, m", [(3, 20), (130, 140)])
def test_the_longest_rows(n, m):
    """2^23 columns, all zeros but a few: exact."""
    k = 1 << 23
    rng = np.random.default_rng(n)
    cols = [0, 5, 127, 128, (1 << 22) + 1, k - 128, k - 1]

    def few(rows):
        codes, values = np.zeros((rows, k), np.uint8), rng.integers(0, 8, (rows, len(cols)))
        codes[:, cols] = np.array([0, 0x38, 0x40, 0x44, 0x48, 0x4a, 0x4c, 0x4e], np.uint8)[values]  # 0 to 7
        return Rows8(rows, k, codes=codes, scales=np.full((rows, k // 128), 127, np.uint8)), values
    (a, x), (w, y) = few(n), few(m)
    np.testing.assert_array_equal(linear8(a, w), x @ y.T)
