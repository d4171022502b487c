"""Matrices in 8 bits written and read back (rows8_write, rows8_read), bit for
bit against the oracle."""

import numpy as np
import pytest

import gpu_helpers as G
from ember_amd import capi
from ember_amd.capi import DeviceArray
from feedforward_helpers import Rows8, ff

pytestmark = pytest.mark.gpu


def write(x, trans=0, pad=0):
    """x (rows, cols), stored with `pad` floats behind each stored row."""
    rows, cols = x.shape
    G.say(f"rows8_write rows={rows} cols={cols} trans={trans} pad={pad}")
    stored = x.T if trans else x
    buf = np.full((stored.shape[0], stored.shape[1] + pad), np.nan, np.float32)
    buf[:, :stored.shape[1]] = stored
    m, dev = Rows8(rows, cols), DeviceArray.from_numpy(buf)
    capi.check(capi.lib().rows8_write(m.view, dev.ptr, buf.shape[1], trans), "rows8_write")
    return m


def read(m, pad=0):
    G.say(f"rows8_read rows={m.rows} cols={m.cols} pad={pad}")
    out = DeviceArray.from_numpy(np.full((m.rows, m.cols + pad), G.SENTINEL))
    capi.check(capi.lib().rows8_read(m.view, out.ptr, m.cols + pad), "rows8_read")
    got = out.numpy()
    assert (got[:, m.cols:] == G.SENTINEL).all()
    return got[:, :m.cols]


def check(x, trans=0, pad=0):
    m = write(x, trans, pad)
    codes, scales = ff.quantise8(x)
    np.testing.assert_array_equal(m.scales.numpy(), scales)
    np.testing.assert_array_equal(m.codes.numpy(), codes)
    with np.errstate(invalid="ignore"):
        np.testing.assert_array_equal(read(m, pad), ff.values8(codes, scales, x.shape[1]).astype(np.float32))


@pytest.mark.parametrize("trans", [0, 1])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 127), (5, 128), (2, 129), (64, 512), (65, 513), (130, 900), (1, 5000), (700, 64)])
def test_sizes(rows, cols, trans):
    rng = np.random.default_rng(rows * cols)
    x = (rng.standard_normal((rows, cols)) * np.exp(2 * rng.standard_normal((rows, cols)))).astype(np.float32)
    for pad in (0, 1, 4):
        check(x, trans, pad)


@pytest.mark.parametrize("trans", [0, 1])
def test_special_values(trans):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((16, 300)).astype(np.float32)
    x[0], x[1] = 0, -0.0
    x[2, 130], x[3, 5], x[4, 299] = np.nan, np.inf, -np.inf
    x[5] *= np.float32(2.0 ** -140)  # denormal numbers
    x[6] = x[6] / np.abs(x[6]).max() * np.float32(2.0 ** 126.9)
    x[7, 3] = 2.0 ** 127
    x[8, :128] = np.resize(np.float32([448, 1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10, -1.0625]), 128)  # ties
    x[9, :128] = 1.75
    x[10, :128] = np.nextafter(np.float32(1.75), np.float32(2))
    x[11] = 2.0 ** -149
    check(x, trans)


@pytest.mark.parametrize("trans", [0, 1])
def test_every_code_and_scale_reads_back(trans):
    codes = np.tile(np.arange(256, dtype=np.uint8), (240, 1))
    scales = np.repeat(np.concatenate((np.arange(8, 247), [255])).astype(np.uint8)[:, None], 4, 1)
    m = Rows8(240, 256, codes=codes, scales=scales)
    with np.errstate(invalid="ignore"):
        want = ff.values8(codes, scales, 256).astype(np.float32)
    np.testing.assert_array_equal(read(m), want)
    fine = np.isfinite(want).all(1)
    assert fine.sum() == 0  # code 127 is in every row
    x = np.where(np.isfinite(want), want, 0)[:, :254]
    x = x[np.abs(x).max(1) < 2.0 ** 127]
    np.testing.assert_array_equal(read(write(x, trans)), x)  # what is held is held again


def test_no_rows():
    m, x = Rows8(0, 70), DeviceArray((70,))
    capi.check(capi.lib().rows8_write(m.view, x.ptr, 70, 0), "rows8_write")
    capi.check(capi.lib().rows8_write(m.view, x.ptr, 70, 1), "rows8_write")
    capi.check(capi.lib().rows8_read(m.view, x.ptr, 70), "rows8_read")
