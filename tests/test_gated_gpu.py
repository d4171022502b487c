"""Gated layers in fp32 (gated_fwd, gated_bwd) against float64, and the whole
backward of one against differences."""

import numpy as np
import pytest

import gpu_helpers as G
from ember_amd import capi
from ember_amd.capi import DeviceArray
from feedforward_helpers import ACT, U, arr, ff, gate_error
from serving_helpers import ptr
from tolerance import gemm_error_bound

pytestmark = pytest.mark.gpu

# (n, hidden, d): one row, odd sizes, whole tiles of each size, k that is cut among workgroups.
SIZES = [(1, 1, 1), (1, 64, 64), (3, 5, 7), (17, 33, 100), (64, 64, 32), (65, 129, 31), (100, 680, 256), (128, 128, 128), (200, 685, 257),
         (256, 256, 64), (300, 1000, 513), (16, 512, 4096), (1024, 512, 512), (1025, 770, 300)]


def forward(x, w, bias, act, want_pre=True, log=None):
    n, d = x.shape
    hidden = w.shape[1] // 2
    G.say(f"gated_fwd n={n} hidden={hidden} d={d} bias={bias is not None} act={act}")
    dx, dw, b = arr(x), arr(w), arr(bias)
    h = DeviceArray.from_numpy(np.full((n, hidden), G.SENTINEL))
    pre = DeviceArray.from_numpy(np.full((n, 2 * hidden), G.SENTINEL)) if want_pre else None
    capi.launch_log_reset()
    rc = capi.lib().gated_fwd(dx.ptr, dw.ptr, ptr(b), h.ptr, ptr(pre), n, hidden, d, ACT[act])
    if log is not None:
        log.extend(capi.launch_log())
    capi.check(rc, "gated_fwd")
    return h.numpy(), None if pre is None else pre.numpy()


def backward(dy, w_down, pre, act, log=None):
    n, d = dy.shape
    hidden = w_down.shape[0]
    G.say(f"gated_bwd n={n} hidden={hidden} d={d} act={act}")
    dev = [arr(a) for a in (dy, w_down, pre)]
    dpre = DeviceArray.from_numpy(np.full((n, 2 * hidden), G.SENTINEL))
    capi.launch_log_reset()
    rc = capi.lib().gated_bwd(*(a.ptr for a in dev), dpre.ptr, n, hidden, d, ACT[act])
    if log is not None:
        log.extend(capi.launch_log())
    capi.check(rc, "gated_bwd")
    return dpre.numpy()


def inputs(n, hidden, d, seed=0):
    rng = np.random.default_rng(n * 7 + hidden * 3 + d + seed)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    return f(n, d), f(d, 2 * hidden) / np.float32(np.sqrt(d)), f(2 * hidden), f(hidden, d) / np.float32(np.sqrt(hidden)), f(n, d)


@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n,hidden,d", SIZES)
def test_forward(n, hidden, d, bias, act):
    x, w, b, _, _ = inputs(n, hidden, d)
    b = b if bias else None
    h, pre = forward(x, w, b, act)
    exact = x.astype(np.float64) @ w + (0 if b is None else b)
    off = gemm_error_bound(x, w) + 2 * U * np.abs(exact)
    assert (np.abs(pre - exact) <= off).all()
    assert np.linalg.norm(pre - exact) <= 32 * U * np.linalg.norm(exact) + 32 * U * np.linalg.norm(np.abs(x).astype(np.float64) @ np.abs(w)) / np.sqrt(d)
    # h is formed of the sums that are kept.
    kept = ff.gate(act, pre.astype(np.float64))
    assert (np.abs(h - kept) <= gate_error(act, pre.astype(np.float64), 0 * off) + 2.0 ** -148).all()
    assert (np.abs(h - ff.gate(act, exact)) <= gate_error(act, exact, off) + 2.0 ** -148).all()
    np.testing.assert_array_equal(forward(x, w, b, act, want_pre=False)[0], h)


def slope_error(act, gate):
    """How far an activation's slope may be off: a few half steps of its terms, of
    which x times the slope of tanh or the logistic function is at most |x|."""
    return 8 * U * (1 + np.abs(gate))


@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("n,hidden,d", SIZES)
def test_backward(n, hidden, d, act):
    x, w, b, w_down, dy = inputs(n, hidden, d, 1)
    pre = (x.astype(np.float64) @ w + b).astype(np.float32)
    got = backward(dy, w_down, pre, act)
    wide = pre.astype(np.float64)
    dh = dy.astype(np.float64) @ w_down.T.astype(np.float64)
    exact = ff.gate_bwd(act, dh, wide)
    off = gemm_error_bound(dy, np.ascontiguousarray(w_down.T))
    value, slope = ff.activate(act, wide[:, :hidden])
    up = wide[:, hidden:]
    tol = np.concatenate(((np.abs(slope) + slope_error(act, wide[:, :hidden])) * np.abs(up) * off + slope_error(act, wide[:, :hidden]) * np.abs(dh * up),
                          (np.abs(value) + 8 * U * np.abs(wide[:, :hidden])) * off + 8 * U * np.abs(wide[:, :hidden] * dh)), 1)
    assert (np.abs(got - exact) <= tol + 4 * U * np.abs(exact) + 2.0 ** -148).all()
    np.testing.assert_array_equal(backward(dy, w_down, pre, act), got)


@pytest.mark.parametrize("act", list(ACT))
def test_far_gates(act):
    """Gates far from zero on both sides, zeros, infinities and NaN."""
    gate = np.float32([0, -0.0, 30, -30, 90, -90, 200, -200, 1e30, -1e30, np.inf, np.nan, 1e-30, 3e38])
    hidden = gate.size
    x, w = np.ones((1, 1), np.float32), np.concatenate((gate, np.full(hidden, 2, np.float32)))[None]
    with np.errstate(all="ignore"):
        h, pre = forward(x, w, None, act)
        want = ff.gate(act, w.astype(np.float64)).astype(np.float32)
        np.testing.assert_array_equal(np.isnan(h[0]), np.isnan(want[0]))
        fine = np.isfinite(want[0])
        assert (h[0][~fine & ~np.isnan(want[0])] == np.inf).all()
        assert (np.abs(h[0] - want[0])[fine] <= 32 * U * np.abs(gate[fine])).all()
        finite = np.isfinite(gate)
        dpre = backward(np.ones((1, 1), np.float32), np.ones((hidden, 1), np.float32), np.where(np.isfinite(w), w, 0), act)[0]
        want = ff.gate_bwd(act, np.ones((1, hidden)), np.where(np.isfinite(w), w, 0).astype(np.float64))[0]
        for half in (dpre[:hidden] - want[:hidden], dpre[hidden:] - want[hidden:]):
            assert (np.abs(half[finite]) <= 32 * U * (1 + np.abs(gate[finite]))).all()


def test_infinite_and_huge_operands():
    """What the split products cannot carry is formed again in fp32."""
    x, w, b, _, _ = inputs(70, 90, 40)
    x[3, 5], x[9, 0], w[7, 100] = np.inf, 1e36, 1e30
    h, pre = forward(x, w, b, "silu")
    with np.errstate(all="ignore"):
        exact = (x.astype(np.float64) @ w + b)
        bad = ~np.isfinite(exact) | (np.abs(exact) > 3e38)
        rest = ~bad
        assert (~np.isfinite(pre[bad])).all()
        wide = np.where(np.isfinite(x), x, 0)
        tol = gemm_error_bound(wide, w) + 2 * U * np.abs(np.where(rest, exact, 0))
        assert (np.abs(pre - exact)[rest] <= tol[rest]).all()
    other = np.ones(70, bool)
    other[[3, 9]] = False
    assert np.isfinite(h[other][:, np.arange(90) != 10]).all()


def test_whole_backward_against_differences():
    """dx, dw, dbias and dw_down of sum(y * dy) for y = h w_down, formed of gated_bwd,
    gemm_ex and col_sum, against central differences of the float64 forward."""
    n, hidden, d, act = 6, 9, 5, "silu"
    x, w, b, w_down, dy = inputs(n, hidden, d, 3)
    h, pre = forward(x, w, b, act)
    L = capi.lib()
    dev = {k: arr(v) for k, v in dict(x=x, w=w, w_down=w_down, dy=dy, pre=pre, h=h).items()}
    new = {k: DeviceArray(s) for k, s in dict(dpre=(n, 2 * hidden), dx=(n, d), dw=(d, 2 * hidden), dw_down=(hidden, d), db=(2 * hidden,)).items()}
    p = lambda k: (dev.get(k) or new[k]).ptr  # noqa: E731
    capi.check(L.gated_bwd(p("dy"), p("w_down"), p("pre"), p("dpre"), n, hidden, d, ACT[act]), "gated_bwd")
    capi.check(L.gemm_ex(p("dpre"), p("w"), p("dx"), 1, n, d, 2 * hidden, 0, 1, None, None, None, 0), "gemm_ex")
    capi.check(L.gemm_ex(p("x"), p("dpre"), p("dw"), 1, d, 2 * hidden, n, 1, 0, None, None, None, 0), "gemm_ex")
    capi.check(L.gemm_ex(p("h"), p("dy"), p("dw_down"), 1, hidden, d, n, 1, 0, None, None, None, 0), "gemm_ex")
    capi.check(L.col_sum(p("dpre"), p("db"), n, 2 * hidden), "col_sum")
    at = dict(x=x, w=w, b=b, w_down=w_down)
    at = {k: v.astype(np.float64) for k, v in at.items()}
    loss = lambda v: (ff.gate(act, v["x"] @ v["w"] + v["b"]) @ v["w_down"] * dy).sum()  # noqa: E731
    for name, grad in (("x", "dx"), ("w", "dw"), ("b", "db"), ("w_down", "dw_down")):
        got = new[grad].numpy()
        for i in np.ndindex(got.shape):
            up, down = dict(at), dict(at)
            up[name], down[name] = at[name].copy(), at[name].copy()
            up[name][i] += 1e-5
            down[name][i] -= 1e-5
            want = (loss(up) - loss(down)) / 2e-5
            assert abs(got[i] - want) <= 2e-5 * (1 + abs(want)), (name, i)


@pytest.mark.parametrize("n,hidden,d", [(5, 12, 8), (70, 200, 36), (300, 260, 2052)])
def test_unaligned(n, hidden, d):
    """Everything 4 bytes off what allocations are aligned to."""
    x, w, b, w_down, dy = inputs(n, hidden, d)
    h, pre = forward(x, w, b, "silu")
    dpre = backward(dy, w_down, pre, "silu")
    off = {k: DeviceArray.from_numpy(np.concatenate(([7.0], v.reshape(-1)))) for k, v in
           dict(x=x, w=w, b=b, w_down=w_down, dy=dy, h=np.zeros_like(h), pre=np.zeros_like(pre), dpre=np.zeros_like(pre)).items()}
    p = {k: v.ptr + 4 for k, v in off.items()}
    G.say(f"gated_fwd, gated_bwd unaligned n={n} hidden={hidden} d={d}")
    capi.check(capi.lib().gated_fwd(p["x"], p["w"], p["b"], p["h"], p["pre"], n, hidden, d, 2), "gated_fwd")
    capi.check(capi.lib().gated_bwd(p["dy"], p["w_down"], p["pre"], p["dpre"], n, hidden, d, 2), "gated_bwd")
    for k, want in (("h", h), ("pre", pre), ("dpre", dpre)):
        got = off[k].numpy()
        assert got[0] == 7
        np.testing.assert_array_equal(got[1:].reshape(want.shape), want)


def test_no_rows():
    p = DeviceArray((64,)).ptr
    capi.check(capi.lib().gated_fwd(p, p, None, p, None, 0, 4, 4, 1), "gated_fwd")
    capi.check(capi.lib().gated_bwd(p, p, p, p, 0, 4, 4, 1), "gated_bwd")


def sweep(act):
    """Gates of all sizes and signs, and the bounds of activation.h in half steps: of
    sigmoid(c x) 5.7, and 1.25 |c x| (1 - sigmoid) where c x is rounded."""
    c = dict(gelu=1.6, silu=1.0)[act]
    rng = np.random.default_rng(11)
    gate = np.concatenate((rng.uniform(-86 / c, 30, 30000), rng.uniform(-2, 2, 9000), -np.exp(rng.uniform(-60, 4, 3000)), np.linspace(-86 / c, 30, 5001),
                           [0.0, 1e30, 3e38])).astype(np.float32)
    x = gate.astype(np.float64)
    small = np.exp(-np.abs(c * x))
    s, rest = np.where(x >= 0, 1, small) / (1 + small), np.where(x >= 0, small, 1) / (1 + small)
    off = (5.7 + (1.25 * np.abs(c * x) * rest if act == "gelu" else 0)) * U
    return gate, c, x, s, rest, off


@pytest.mark.parametrize("act", list(ACT))
def test_the_gate_is_near_in_relative_terms(act):
    """act(gate) * 1 within the sigmoid's bound and one rounding of itself, far below 0 too."""
    gate, _, x, s, _, off = sweep(act)
    h, pre = forward(gate[:, None], np.float32([[1, 0]]), np.float32([0, 1]), act)
    np.testing.assert_array_equal(pre, np.stack((gate, np.ones_like(gate)), 1))
    assert (np.abs(h[:, 0] - x * s) <= (off + 1.1 * U) * np.abs(x * s) + 2.0 ** -149).all()


@pytest.mark.parametrize("act", list(ACT))
def test_the_gates_gradient_is_near(act):
    """Both halves of dpre for dh = up = 1: the value as above; the slope is s + c (v (1 -
    s)), where v = x s carries s's bound and a rounding, 1 - s what s is off by and a
    rounding, and two products and c round; the sum once more."""
    gate, c, x, s, rest, off = sweep(act)
    one = np.ones((len(gate), 1), np.float32)
    dpre = backward(one, np.ones((1, 1), np.float32), np.stack((gate, one[:, 0]), 1), act)
    slope = s + c * x * s * rest
    tol = off * s + c * np.abs(x) * s * ((off + 4.3 * U) * rest + off * s) + 1.1 * U * np.abs(slope)
    assert (np.abs(dpre[:, 0] - slope) <= 1.001 * tol + 2.0 ** -148).all()
    assert (np.abs(dpre[:, 1] - x * s) <= (off + 1.1 * U) * np.abs(x * s) + 2.0 ** -149).all()


@pytest.mark.parametrize("act", list(ACT))
def test_gates_past_the_sigmoids_range(act):
    """Between the result and 0 from c gate = -86 on down; -0 or NaN, never anything else."""
    c = dict(gelu=1.6, silu=1.0)[act]
    gate = -np.concatenate((np.linspace(86, 110, 4001), [120, 150, 200, 1e4, 1e30, 3e38])).astype(np.float32) / np.float32(c)
    h, _ = forward(gate[:, None], np.float32([[1, 0]]), np.float32([0, 1]), act)
    x = gate.astype(np.float64)
    exact = x * np.exp(c * x)  # within 2^-124 of itself
    assert (h[:, 0] <= 0).all() and (h[:, 0] >= exact * (1 + 300 * U) - 2.0 ** -148).all()
    assert (exact[h[:, 0] == 0] > -(2.0 ** -118)).all()
