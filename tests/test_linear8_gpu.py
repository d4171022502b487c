"""Products of 8-bit matrices (linear8_fwd) and gated layers of them
(gated8_fwd), against float64 over the values that the codes stand for."""

import numpy as np
import pytest

from feedforward_helpers import ACT, Rows8, U, check_held, ff, gate_error, gated8, linear8, product, sum_error

pytestmark = pytest.mark.gpu

# (n, m, k): one row to many, odd columns, k of one group, of a part of one and of many.
SIZES = [(1, 1, 1), (1, 16, 128), (2, 33, 130), (15, 100, 1000), (16, 48, 512), (17, 257, 127), (31, 64, 4096), (33, 130, 640), (64, 200, 129),
         (65, 96, 256), (100, 1000, 200), (129, 129, 1025), (256, 256, 384), (300, 520, 777), (513, 40, 2048)]


def operands(n, m, k, seed=0):
    rng = np.random.default_rng(n * 1000003 + m * 1009 + k + seed)
    a = (rng.standard_normal((n, k)) * np.exp(0.7 * rng.standard_normal(k))).astype(np.float32)
    w = (rng.standard_normal((m, k)) / np.sqrt(k) * np.exp(0.7 * rng.standard_normal((m, 1)))).astype(np.float32)
    return Rows8.of(a), Rows8.of(w), rng


def check_product(out, exact, reach, k, more=0):
    np.testing.assert_array_equal(np.isnan(out), np.isnan(exact))
    fine = np.isfinite(exact)
    assert (np.abs(out - exact)[fine] <= (sum_error(reach, k) + 2 * U * np.abs(exact) + more)[fine] + 2.0 ** -148).all()
    if fine.any():  # independent roundings of a few steps each
        assert np.linalg.norm((out - exact)[fine]) <= 32 * U * np.linalg.norm(exact[fine]) + 32 * U * np.linalg.norm(reach[fine]) / np.sqrt(k)


@pytest.mark.parametrize("n,m,k", SIZES)
def test_product(n, m, k):
    a, w, _ = operands(n, m, k)
    out = linear8(a, w)
    check_product(out, *product(a, w), k)
    np.testing.assert_array_equal(linear8(a, w), out)


@pytest.mark.parametrize("n,m,k", SIZES)
@pytest.mark.parametrize("parts", ["bias", "residual", "both", "gelu"])
def test_epilogue(n, m, k, parts):
    a, w, rng = operands(n, m, k, 1)
    bias = rng.standard_normal(m).astype(np.float32) if parts != "residual" else None
    residual = rng.standard_normal((n, m)).astype(np.float32) if parts != "bias" else None
    act = int(parts == "gelu")
    exact, reach = product(a, w)
    exact = exact + (0 if bias is None else bias)
    off = sum_error(reach, k) + 2 * U * np.abs(exact)
    if act:
        off, exact = 1.2 * off + 8 * U * np.abs(exact), ff.activate("gelu", exact)[0]
    exact = exact + (0 if residual is None else residual)
    out = linear8(a, w, bias, residual, act)
    assert (np.abs(out - exact) <= off + 2 * U * np.abs(exact) + 2.0 ** -148).all()


@pytest.mark.parametrize("n", [3, 40, 200])
def test_exact_where_fp32_is(n):
    """Small whole numbers: every sum is exact, in any order."""
    rng = np.random.default_rng(n)
    a, w = rng.integers(-15, 16, (n, 600)).astype(np.float32), rng.integers(-15, 16, (300, 600)).astype(np.float32)
    np.testing.assert_array_equal(linear8(Rows8.of(a), Rows8.of(w)), a @ w.T)


@pytest.mark.parametrize("n", [1, 20, 64, 300])
def test_terms_far_below_the_largest(n):
    """Sums whose large terms cancel, so that what is left are terms 2^-16 of them."""
    rng = np.random.default_rng(n)
    a = rng.integers(1, 16, (n, 256)).astype(np.float32) * 2.0 ** -8
    w = rng.integers(1, 16, (96, 256)).astype(np.float32)
    a[:, 3:128:16], w[:, 3:128:16] = 240, 15  # first parts of a group large, and again with the other sign
    a[:, 4:128:16], w[:, 4:128:16] = -240, 15
    exact = a.astype(np.float64) @ w.T.astype(np.float64)
    np.testing.assert_array_equal(linear8(Rows8.of(a), Rows8.of(w)), exact)


@pytest.mark.parametrize("n", [2, 30, 150])
def test_all_codes_and_scales(n):
    rng = np.random.default_rng(n + 5)
    codes = lambda r: np.where(rng.random((r, 512)) < 0.5, 0, 128).astype(np.uint8) + rng.integers(0, 127, (r, 512)).astype(np.uint8)  # noqa: E731
    a = Rows8(n, 512, codes=codes(n), scales=rng.integers(60, 120, (n, 4)).astype(np.uint8))
    w = Rows8(70, 512, codes=codes(70), scales=rng.integers(100, 180, (70, 4)).astype(np.uint8))
    check_product(linear8(a, w), *product(a, w), 512)


@pytest.mark.parametrize("n", [2, 40, 150])
def test_smallest_and_largest_scales(n):
    """Values down to 2^-128, below fp32's smallest normal number, times ones near
    its largest, and the other way round."""
    rng = np.random.default_rng(n + 7)
    codes = lambda r: rng.integers(0, 127, (r, 256)).astype(np.uint8)  # noqa: E731
    low = lambda r: rng.integers(8, 11, (r, 4)).astype(np.uint8)  # noqa: E731
    high = lambda r: rng.integers(240, 246, (r, 4)).astype(np.uint8)  # noqa: E731
    for x, y in ((low, high), (high, low)):
        a, w = Rows8(n, 256, codes=codes(n), scales=x(n)), Rows8(70, 256, codes=codes(70), scales=y(70))
        check_product(linear8(a, w), *product(a, w), 256)
    # The smallest codes alone: 2^-9 of the smallest scale.
    one, ones = np.ones((n, 128), np.uint8), np.full((33, 128), 0x38, np.uint8)  # 2^-9 and 1
    a, w = Rows8(n, 128, codes=one, scales=np.full((n, 4), 8, np.uint8)), Rows8(33, 128, codes=ones, scales=np.full((33, 4), 246, np.uint8))
    np.testing.assert_array_equal(linear8(a, w), 128 * 2.0 ** -9)


@pytest.mark.parametrize("n", [4, 50, 260])
def test_nan_reaches_its_row_and_column_only(n):
    a, w, _ = operands(n, 40, 300)
    codes, scales = a.bytes()
    codes[1, 17] = 127
    scales[n - 1, 2] = 255
    a = Rows8(n, 300, codes=codes, scales=scales)
    codes, scales = w.bytes()
    codes[5, 299], scales[20, 0] = 255, 255
    w = Rows8(40, 300, codes=codes, scales=scales)
    out = linear8(a, w)
    want = np.zeros((n, 40), bool)
    want[[1, n - 1]], want[:, [5, 20]] = True, True
    np.testing.assert_array_equal(np.isnan(out), want)
    exact, reach = product(a, w)
    check_product(out, exact, reach, 300)


def test_out_may_be_residual():
    from ember_amd import capi
    from ember_amd.capi import DeviceArray
    for n in (5, 200):
        a, w, rng = operands(n, 72, 260)
        r = rng.standard_normal((n, 72)).astype(np.float32)
        dev = DeviceArray.from_numpy(r)
        capi.check(capi.lib().linear8_fwd(a.view, w.view, None, dev.ptr, dev.ptr, 0), "linear8_fwd")
        np.testing.assert_array_equal(dev.numpy(), linear8(a, w, None, r))


@pytest.mark.parametrize("n", [2, 100])
def test_unaligned_out_bias_and_residual(n):
    from ember_amd import capi
    from ember_amd.capi import DeviceArray
    a, w, rng = operands(n, 64, 128)
    bias, r = rng.standard_normal(64).astype(np.float32), rng.standard_normal((n, 64)).astype(np.float32)
    dev = [DeviceArray.from_numpy(np.concatenate(([7.0], x.reshape(-1)))) for x in (bias, r, np.zeros((n, 64)))]
    capi.check(capi.lib().linear8_fwd(a.view, w.view, *(d.ptr + 4 for d in dev), 0), "linear8_fwd")
    got = dev[2].numpy()
    assert got[0] == 7
    np.testing.assert_array_equal(got[1:].reshape(n, 64), linear8(a, w, bias, r))


def test_no_rows_or_columns():
    one = Rows8(1, 20, fill=0)
    assert linear8(Rows8(0, 20), one).size == 0 and linear8(one, Rows8(0, 20)).size == 0
    assert gated8(Rows8(0, 20), Rows8(2, 20), None, "silu").codes.n == 0


@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n,hidden,k", [(1, 1, 1), (1, 128, 128), (2, 130, 200), (16, 300, 1000), (17, 64, 2048), (33, 1000, 129), (64, 257, 640),
                                        (65, 128, 256), (130, 385, 500), (257, 640, 1200)])
def test_gated(n, hidden, k, bias, act):
    a, w, rng = operands(n, 2 * hidden, k, 2)
    b = rng.standard_normal(2 * hidden).astype(np.float32) if bias else None
    h = gated8(a, w, b, act)
    pre, reach = product(a, w)
    pre = pre + (0 if b is None else b)
    exact = ff.gate(act, pre)
    check_held(h, exact, gate_error(act, pre, sum_error(reach, k) + 2 * U * np.abs(pre)))
    again = gated8(a, w, b, act)
    for x, y in zip(again.bytes(), h.bytes()):
        np.testing.assert_array_equal(x, y)


@pytest.mark.parametrize("n", [3, 70, 300])
def test_gated_nan_marks_its_groups(n):
    a, w, _ = operands(n, 2 * 300, 256)
    codes, scales = a.bytes()
    codes[2, 100] = 127
    a = Rows8(n, 256, codes=codes, scales=scales)
    codes, scales = w.bytes()
    scales[300 + 200, 1] = 255  # a row of the other projection: column 200, in group 1
    w = Rows8(600, 256, codes=codes, scales=scales)
    h = gated8(a, w, None, "gelu")
    s = h.bytes()[1]
    assert (s[2, :3] == 255).all() and (s[:, 1] == 255).all() and (s[:, 3] == 127).all()
    assert (np.delete(s[:, [0, 2]], 2, 0) != 255).all()
    assert (h.bytes()[0][:, 128:256] == 0).all()


@pytest.mark.parametrize("n,m", [(1, 33), (16, 20), (7, 4096), (2, 4097)])
@pytest.mark.parametrize("k", [1024, 1025, 1152, 1300, 2048, 2177, 4224])
def test_runs_of_k_that_few_waves_share(n, m, k):
    """8 groups of k and 9, 11, 16, 18 and 33, of which two and four waves have uneven runs, some none."""
    a, w, _ = operands(n, m, k, 9)
    check_product(linear8(a, w), *product(a, w), k)


@pytest.mark.parametrize("n,m,k", [(40, 5101, 300), (100, 40, 4089), (257, 3001, 2100), (500, 4000, 384), (1500, 4001, 100), (4000, 2049, 640)])
def test_out_may_be_residual_in_every_kernel(n, m, k):
    from ember_amd import capi
    from ember_amd.capi import DeviceArray
    a, w, rng = operands(n, m, k, 12)
    bias, r = rng.standard_normal(m).astype(np.float32), rng.standard_normal((n, m)).astype(np.float32)
    dev, b = DeviceArray.from_numpy(r), DeviceArray.from_numpy(bias)
    capi.check(capi.lib().linear8_fwd(a.view, w.view, b.ptr, dev.ptr, dev.ptr, 1), "linear8_fwd")
    np.testing.assert_array_equal(dev.numpy(), linear8(a, w, bias, r, 1))
