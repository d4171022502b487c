"""RMS norm (rmsnorm_fwd, rmsnorm_fwd8, rmsnorm_bwd) against float64."""

import numpy as np
import pytest

import gpu_helpers as G
from ember_amd import capi
from ember_amd.capi import DeviceArray
from feedforward_helpers import Rows8, arr, check_held, ff
from serving_helpers import U, ptr

pytestmark = pytest.mark.gpu

# One wave to a row to 1024, four to 4096, sixteen to 16384; rows that fill no chunk.
SIZES = [(1, 4), (5, 60), (3, 128), (9, 516), (4, 1024), (7, 1028), (2, 4096), (3, 4100), (2, 16384), (1, 12000), (70, 260)]


def norm(x, residual, gamma, eps=1e-5, want_sum=True, want_rstd=True, inplace=False):
    rows, d = x.shape
    G.say(f"rmsnorm_fwd rows={rows} d={d} residual={residual is not None} inplace={inplace}")
    dx, r, g = arr(x), arr(residual), arr(gamma)
    s = dx if inplace else DeviceArray.from_numpy(np.full(x.shape, G.SENTINEL)) if want_sum else None
    y = (r if r is not None else DeviceArray(x.shape)) if inplace else DeviceArray.from_numpy(np.full(x.shape, G.SENTINEL))
    rstd = DeviceArray((rows,)) if want_rstd else None
    capi.check(capi.lib().rmsnorm_fwd(dx.ptr, ptr(r), g.ptr, ptr(s), y.ptr, ptr(rstd), rows, d, eps), "rmsnorm_fwd")
    return y.numpy(), None if s is None else s.numpy(), None if rstd is None else rstd.numpy()


def norm8(x, residual, gamma, eps=1e-5, want_sum=True):
    rows, d = x.shape
    G.say(f"rmsnorm_fwd8 rows={rows} d={d} residual={residual is not None}")
    dx, r, g, y = arr(x), arr(residual), arr(gamma), Rows8(rows, d)
    s = DeviceArray.from_numpy(np.full(x.shape, G.SENTINEL)) if want_sum else None
    capi.check(capi.lib().rmsnorm_fwd8(dx.ptr, ptr(r), g.ptr, ptr(s), y.view, eps), "rmsnorm_fwd8")
    return y, None if s is None else s.numpy()


def inputs(rows, d, residual, seed=0, size=1.0):
    rng = np.random.default_rng(1000 * rows + d + seed)
    x = (size * rng.standard_normal((rows, d)) * np.exp(0.5 * rng.standard_normal(d))).astype(np.float32)
    r = (size * rng.standard_normal((rows, d))).astype(np.float32) if residual else None
    return x, r, (1 + 0.3 * rng.standard_normal(d)).astype(np.float32)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,d", SIZES)
def test_forward(rows, d, residual):
    x, r, gamma = inputs(rows, d, residual)
    s = x if r is None else x + r
    y, got, rstd = norm(x, r, gamma)
    ry, rr = ff.rmsnorm_fwd(s, gamma, 1e-5)
    np.testing.assert_array_equal(got, s)
    # One rounding each; the double sums' own are 2^-29 of it.
    assert (np.abs(y - ry) <= U * (1 + 2.0 ** -20) * np.abs(ry)).all()
    assert (np.abs(rstd - rr) <= U * (1 + 2.0 ** -20) * rr).all()
    same, none, _ = norm(x, r, gamma, want_sum=False, want_rstd=False)
    np.testing.assert_array_equal(same, y)
    assert none is None


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,d", SIZES)
def test_forward_in_8_bits_is_the_norm_then_rounded(rows, d, residual):
    x, r, gamma = inputs(rows, d, residual)
    y, _, _ = norm(x, r, gamma)
    held, s = norm8(x, r, gamma)
    for got, want in zip(held.bytes(), ff.quantise8(y)):
        np.testing.assert_array_equal(got, want)
    np.testing.assert_array_equal(s, x if r is None else x + r)
    check_held(held, ff.rmsnorm_fwd(s, gamma, 1e-5)[0], U * np.abs(y) * 2)
    again, none = norm8(x, r, gamma, want_sum=False)
    np.testing.assert_array_equal(again.bytes()[0], held.bytes()[0])


@pytest.mark.parametrize("residual", [False, True])
def test_in_place(residual):
    x, r, gamma = inputs(6, 1540, residual)
    y, s, rstd = norm(x, r, gamma)
    if residual:  # the sum over x, y over the residual
        y2, s2, rstd2 = norm(x, r, gamma, inplace=True)
        np.testing.assert_array_equal(s2, s)
    else:  # y over x
        dx, g = arr(x), arr(gamma)
        capi.check(capi.lib().rmsnorm_fwd(dx.ptr, None, g.ptr, None, dx.ptr, None, 6, 1540, 1e-5), "rmsnorm_fwd")
        y2 = dx.numpy()
    np.testing.assert_array_equal(y2, y)


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e12, 1e30])
def test_sizes_whose_squares_leave_fp32(size):
    x, _, gamma = inputs(3, 640, False, size=size)
    y, _, rstd = norm(x, None, gamma, eps=0.0)
    ry, rr = ff.rmsnorm_fwd(x, gamma, 0.0)
    assert (np.abs(y - ry) <= U * (1 + 2.0 ** -20) * np.abs(ry)).all() and np.isfinite(y).all()
    assert (np.abs(rstd - rr) <= U * (1 + 2.0 ** -20) * rr).all()


def test_rows_of_zeros_infinities_and_nan():
    x, _, gamma = inputs(5, 260, False)
    x[0], x[1, 7], x[2, 200], x[3, 3] = 0, np.inf, np.nan, -np.inf
    y, _, _ = norm(x, None, gamma)
    assert (y[0] == 0).all() and np.isnan(y[2]).all()
    for row, at in ((1, 7), (3, 3)):  # 1/sqrt(infinity) is 0, and times infinity NaN
        assert np.isnan(y[row, at]) and (np.delete(y[row], at) == 0).all()
    assert np.isfinite(y[4]).all()
    held, _ = norm8(x, None, gamma)
    v = held.values()
    assert (v[0] == 0).all() and np.isnan(v[2]).all() and np.isnan(v[1, :128]).all() and (v[1, 128:] == 0).all()
    np.testing.assert_array_equal(v[4], ff.values8(*ff.quantise8(y[4:5]), 260)[0])


@pytest.mark.parametrize("dres", [False, True])
@pytest.mark.parametrize("rows,d", SIZES + [(1000, 512), (300, 2052), (33, 8192)])
def test_backward(rows, d, dres):
    s, more, gamma = inputs(rows, d, dres, seed=7)
    dy = np.random.default_rng(d).standard_normal(s.shape).astype(np.float32)
    rstd = ff.rmsnorm_fwd(s, gamma, 1e-5)[1].astype(np.float32)
    dx, dgamma = backward(s, gamma, rstd, dy, more)
    rdx, rdg = ff.rmsnorm_bwd(s, gamma, rstd, dy, more)
    xhat, g = s.astype(np.float64) * rstd[:, None], dy.astype(np.float64) * gamma
    mean = np.abs(g * xhat).mean(-1, keepdims=True)
    # The mean is a sum of at most 16 elements a lane, 6 steps over a wave and 16 waves, of
    # products of two roundings each; the rest is a few roundings of each term.
    tol = rstd[:, None] * (8 * U * (np.abs(g) + np.abs(xhat) * mean) + 48 * U * np.abs(xhat) * mean) + 4 * U * np.abs(rdx) + (0 if more is None else 4 * U * np.abs(more))
    assert (np.abs(dx - rdx) <= tol + 1e-40).all()
    assert (np.abs(dgamma - rdg) <= (rows + 8) * U * np.abs(dy * xhat).sum(0)).all()
    # Independent roundings: far fewer than rows steps in the 2-norm.
    assert np.linalg.norm(dgamma - rdg) <= 32 * U * np.linalg.norm(np.sqrt(((dy * xhat) ** 2).sum(0))) + 1e-30
    again = backward(s, gamma, rstd, dy, more)
    np.testing.assert_array_equal(again[0], dx)
    np.testing.assert_array_equal(again[1], dgamma)


def backward(s, gamma, rstd, dy, dres):
    rows, d = s.shape
    G.say(f"rmsnorm_bwd rows={rows} d={d} dres={dres is not None}")
    dev = [arr(a) for a in (s, gamma, rstd, dy)]
    r, dx, dg = arr(dres), DeviceArray.from_numpy(np.full(s.shape, G.SENTINEL)), DeviceArray.from_numpy(np.full(d, G.SENTINEL))
    capi.check(capi.lib().rmsnorm_bwd(*(a.ptr for a in dev), ptr(r), dx.ptr, dg.ptr, rows, d), "rmsnorm_bwd")
    return dx.numpy(), dg.numpy()


def test_no_rows():
    gamma, dg, y = arr(np.ones(8)), arr(np.full(8, 5.0)), Rows8(0, 8)
    p = DeviceArray((1,)).ptr
    L = capi.lib()
    capi.check(L.rmsnorm_fwd(p, None, gamma.ptr, None, p, None, 0, 8, 1e-5), "rmsnorm_fwd")
    capi.check(L.rmsnorm_fwd8(p, None, gamma.ptr, None, y.view, 1e-5), "rmsnorm_fwd8")
    capi.check(L.rmsnorm_bwd(p, gamma.ptr, p, p, None, p, dg.ptr, 0, 8), "rmsnorm_bwd")
    assert (dg.numpy() == 0).all()


@pytest.mark.parametrize("rows,d,run", [((1 << 22) + 5, 4, 1024), ((1 << 19) + 3, 1028, 512), ((1 << 17) + 1, 4100, 512)])
def test_gradient_of_gamma_of_many_rows(rows, d, run):
    """The error of a column's sum does not grow with the rows.  All terms dy * xhat are
    t = 1 + 0.45 of the last place of a sum of run / 2 to run, which is cut off whenever t
    is added to one: run terms one by one would be off by run / 5 half steps.  At most 32
    terms are summed in 32 bits, then rounded, the four waves' sums added, and 8, 15 and
    7 sums of those: 66 half steps."""
    t = np.float32(1 + 0.45 * run * 2.0 ** -24)
    ones, rstd, gamma = arr(np.ones((rows, d), np.float32)), arr(np.full(rows, t, np.float32)), arr(np.ones(d, np.float32))
    dx, dg = DeviceArray((rows, d)), DeviceArray.from_numpy(np.full(d, G.SENTINEL))
    G.say(f"rmsnorm_bwd rows={rows} d={d}")
    capi.check(capi.lib().rmsnorm_bwd(ones.ptr, gamma.ptr, rstd.ptr, ones.ptr, None, dx.ptr, dg.ptr, rows, d), "rmsnorm_bwd")
    exact = rows * float(t)
    assert (np.abs(dg.numpy() - exact) <= 66 * U * exact).all()


@pytest.mark.parametrize("rows,d", [(5, 60), (70, 1024), (3, 4096), (40, 1540), (3, 16384)])
def test_calls_that_write_over_an_input(rows, d):
    """dx over dres; the sum in 8 bits' forward over x, and over the residual."""
    s, more, gamma = inputs(rows, d, True, seed=13)
    dy = np.random.default_rng(d).standard_normal(s.shape).astype(np.float32)
    rstd = ff.rmsnorm_fwd(s, gamma, 1e-5)[1].astype(np.float32)
    dx, dgamma = backward(s, gamma, rstd, dy, more)
    dev, over, dg = [arr(a) for a in (s, gamma, rstd, dy)], arr(more), DeviceArray((d,))
    capi.check(capi.lib().rmsnorm_bwd(*(a.ptr for a in dev), over.ptr, over.ptr, dg.ptr, rows, d), "rmsnorm_bwd")
    np.testing.assert_array_equal(over.numpy(), dx)
    np.testing.assert_array_equal(dg.numpy(), dgamma)
    held, total = norm8(s, more, gamma)
    for which in (0, 1):
        pair, g, y = [arr(s), arr(more)], arr(gamma), Rows8(rows, d)
        capi.check(capi.lib().rmsnorm_fwd8(pair[0].ptr, pair[1].ptr, g.ptr, pair[which].ptr, y.view, 1e-5), "rmsnorm_fwd8")
        np.testing.assert_array_equal(pair[which].numpy(), total)
        for got, want in zip(y.bytes(), held.bytes()):
            np.testing.assert_array_equal(got, want)
