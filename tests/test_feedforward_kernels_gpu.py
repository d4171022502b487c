"""Every kernel that products of 8-bit matrices and gated layers choose among, by
the launch log, at odd sizes: each shape of tile, whole sums of k and parts of it
that end anywhere, and each width of the kernel for few rows."""

import numpy as np
import pytest

from feedforward_helpers import ACT, Rows8, U, check_held, ff, gate_error, gated8, linear8, product, sum_error
from test_gated_gpu import backward, forward, inputs, slope_error
from test_linear8_gpu import check_product, operands
from tolerance import gemm_error_bound

pytestmark = pytest.mark.gpu

AHEAD, TILES, LARGE, REDUCE = "linear8_tiles128_ahead", "linear8_tiles128", "linear8_tiles256", "linear8_reduce"
PRODUCTS = [
    ([TILES], 1500, 4001, 100), ([TILES], 1505, 4000, 256), ([TILES], 1500, 4000, 600),
    ([AHEAD], 500, 4000, 384), ([AHEAD], 500, 3999, 512), ([AHEAD], 500, 4000, 520), ([AHEAD], 499, 4000, 700),
    ([AHEAD], 500, 4000, 896), ([AHEAD], 500, 4001, 1024), ([AHEAD], 512, 4000, 1100),
    ([AHEAD, REDUCE], 100, 40, 4089), ([AHEAD, REDUCE], 100, 41, 5120), ([AHEAD, REDUCE], 257, 3001, 2100), ([AHEAD, REDUCE], 257, 3000, 2432),
    ([TILES, REDUCE], 257, 3000, 3200), ([TILES, REDUCE], 300, 3001, 5100),
    ([TILES], 128, 50000, 130), ([AHEAD], 64, 20001, 1000), ([LARGE], 2049, 4100, 500), ([LARGE], 4000, 2049, 640), ([LARGE], 5000, 2001, 1000),
]
FEW = [(1, 40, 5000), (16, 48, 4096), (9, 4000, 4500), (5, 10201, 130), (9, 10200, 130), (16, 5101, 200), (20, 10200, 300), (32, 5100, 640), (33, 5100, 129),
       (48, 10201, 200), (64, 10200, 130), (50, 5101, 1000), (70, 900, 1300)]


@pytest.mark.parametrize("kernels,n,m,k", PRODUCTS + [(["linear8_few"], *s) for s in FEW])
def test_products(kernels, n, m, k):
    a, w, rng = operands(n, m, k, 4)
    log = []
    out = linear8(a, w, log=log)
    assert log == kernels
    exact, reach = product(a, w)
    check_product(out, exact, reach, k)
    bias, residual = rng.standard_normal(m).astype(np.float32), rng.standard_normal((n, m)).astype(np.float32)
    for act in (0, 1):
        sums = exact + bias
        off = sum_error(reach, k) + 2 * U * np.abs(sums)
        if act:
            off, sums = 1.2 * off + 8 * U * np.abs(sums), ff.activate("gelu", sums)[0]
        sums += residual
        assert (np.abs(linear8(a, w, bias, residual, act) - sums) <= off + 2 * U * np.abs(sums) + 2.0 ** -148).all()


GATED = [
    (["gated8_tiles128"], 1000, 2001, 100), (["gated8_tiles128"], 640, 3000, 130), (["gated8_tiles128"], 1000, 2000, 384), (["gated8_tiles128"], 999, 2000, 1000),
    (["gated8_tiles256"], 1500, 3001, 128), (["gated8_tiles256"], 1025, 4000, 200), (["gated8_tiles256"], 2000, 2999, 640),
    ([AHEAD, "gated8_reduce"], 130, 200, 4096), (["gated8_few", "rows8_write"], 130, 200, 2048), ([AHEAD, "gated8_reduce"], 65, 41, 3100), ([AHEAD, "gated8_reduce"], 257, 4000, 760),
    ([TILES, "gated8_reduce"], 513, 2000, 2940), ([TILES, "gated8_reduce"], 257, 4001, 4096),
    *((["gated8_few", "rows8_write"], *s) for s in [(1, 500, 5000), (16, 130, 400), (20, 1000, 300), (40, 8200, 130), (64, 8300, 257), (33, 129, 1000)]),
]


@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("kernels,n,hidden,k", GATED)
def test_gated_layers(kernels, n, hidden, k, act):
    a, w, rng = operands(n, 2 * hidden, k, 5)
    b = rng.standard_normal(2 * hidden).astype(np.float32)
    log = []
    h = gated8(a, w, b, act, log)
    assert log == kernels
    pre, reach = product(a, w)
    pre = pre + b
    check_held(h, ff.gate(act, pre), gate_error(act, pre, sum_error(reach, k) + 2 * U * np.abs(pre)))


# (n, hidden, d) and whether the forward and the backward add parts of their sums:
# tiles of 64, 128 and 256 rows with each.
FP32 = [(200, 685, 257, False, True), (700, 600, 3001, True, True), (1500, 1100, 200, False, False), (2049, 2101, 130, False, False),
        (2500, 1300, 2100, True, False), (2049, 1401, 4100, True, True), (4100, 4000, 90, False, False),
        (2000, 4001, 300, False, False), (4095, 4095, 130, False, False)]


@pytest.mark.parametrize("n,hidden,d,fwd_parts,bwd_parts", FP32)
def test_gated_layers_in_fp32(n, hidden, d, fwd_parts, bwd_parts):
    x, w, b, w_down, dy = inputs(n, hidden, d, 6)
    log = []
    h, pre = forward(x, w, b, "silu", log=log)
    assert log == ["gated_fwd", "gate_fwd_reduce"][:1 + fwd_parts]
    exact = x.astype(np.float64) @ w + b
    off = gemm_error_bound(x, w) + 2 * U * np.abs(exact)
    assert (np.abs(pre - exact) <= off).all()
    wide = pre.astype(np.float64)
    assert (np.abs(h - ff.gate("silu", wide)) <= gate_error("silu", wide, 0 * off) + 2.0 ** -148).all()
    log = []
    got = backward(dy, w_down, pre, "silu", log=log)
    assert log == ["gated_bwd", "gate_bwd_reduce"][:1 + bwd_parts]
    dh = dy.astype(np.float64) @ w_down.T.astype(np.float64)
    off = gemm_error_bound(dy, np.ascontiguousarray(w_down.T))
    gate, up = wide[:, :hidden], wide[:, hidden:]
    value, slope = ff.activate("silu", gate)
    tol = np.concatenate(((np.abs(slope) + slope_error("silu", gate)) * np.abs(up) * off + slope_error("silu", gate) * np.abs(dh * up),
                          (np.abs(value) + 8 * U * np.abs(gate)) * off + 8 * U * np.abs(gate * dh)), 1)
    want = ff.gate_bwd("silu", dh, wide)
    assert (np.abs(got - want) <= tol + 4 * U * np.abs(want) + 2.0 ** -148).all()
