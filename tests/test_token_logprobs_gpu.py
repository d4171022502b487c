"""token_logprobs and its gradient through the C ABI against float64: one row
and many, classes from 1 to several segments of a row, ties, infinities and
NaN, padded places, and the gradient against differences."""

import numpy as np
import pytest

import gpu_helpers as G
from ember_amd import capi
from ember_amd.capi import DeviceArray
from oracle import serving
from serving_helpers import U, ints, ptr

pytestmark = pytest.mark.gpu


def padded(x, pad):
    """x's rows with `pad` further floats each, on the device."""
    buf = np.full((x.shape[0], x.shape[1] + pad), G.SENTINEL, np.float32)
    buf[:, :x.shape[1]] = x
    return DeviceArray.from_numpy(buf)


def score(x, tokens, top, pad=0, only_logp=False):
    rows, classes = x.shape
    G.say(f"token_logprobs rows={rows} classes={classes} top={top} pad={pad}")
    dx, tk = padded(x, pad), ints(tokens)
    logp, lse, ent = (DeviceArray((rows,)) for _ in range(3))
    ids, best = ints(np.full((rows, top), -7)) if top else None, DeviceArray((rows, top)) if top else None
    rc = capi.lib().token_logprobs(dx.ptr, classes + pad, tk.ptr, rows, classes, logp.ptr, None if only_logp else lse.ptr,
                                   None if only_logp else ent.ptr, ptr(ids), ptr(best), top)
    capi.check(rc, "token_logprobs")
    if only_logp:
        return logp.numpy()
    return (*(a.numpy() for a in (logp, lse, ent)), ids.numpy() if top else None, best.numpy() if top else None)


def gradient(x, tokens, lse, ent, d_logp, d_ent, pad=0, out_pad=0, in_place=False):
    rows, classes = x.shape
    G.say(f"token_logprobs_bwd rows={rows} classes={classes} pad={pad}")
    dx, tk = padded(x, pad), ints(tokens)
    out = dx if in_place else padded(np.zeros_like(x), out_pad)
    dev = [None if a is None else DeviceArray.from_numpy(a) for a in (lse, ent, d_logp, d_ent)]
    stride = classes + (pad if in_place else out_pad)
    capi.check(capi.lib().token_logprobs_bwd(dx.ptr, classes + pad, tk.ptr, *(ptr(a) for a in dev), out.ptr, stride, rows, classes),
               "token_logprobs_bwd")
    full = out.numpy()
    assert (full[:, classes:] == G.SENTINEL).all()
    return full[:, :classes]


def check(x, tokens, top, **more):
    """Within the roundings of the sums: x - m is off by half a step of up to the
    range r of a row; exp and log by a step; the sum over `classes` terms is
    taken in 32 per thread and a tree of 8 + 2 log2 levels, 64 roundings at
    most before the joins.  So ln s is off by (r + 64 + 2 log2(classes)) half
    steps, relative to s where one term leads, and the entropy, a mean of x - m,
    by as many times the range."""
    rows, classes = x.shape
    logp, lse, ent, ids, best = score(x, tokens, top, **more)
    rp, rl, re, ri, rb = serving.token_logprobs(x, tokens, top)
    r = np.ptp(x.astype(np.float64), -1)
    off = U * (r + 64 + 2 * np.log2(classes + 1))
    assert (np.abs(logp - rp) <= off + 2 * U * np.abs(rp)).all()
    assert (np.abs(lse - rl) <= off + 2 * U * (np.abs(rl) + np.abs(x).max(-1))).all()
    assert (np.abs(ent - re) <= 2 * off * (1 + np.minimum(r, 40))).all()
    if top:
        np.testing.assert_array_equal(ids, ri)
        assert (np.abs(best - rb) <= off[:, None] + 2 * U * np.abs(rb)).all()
    return logp, lse, ent


@pytest.mark.parametrize("classes", [1, 2, 3, 31, 64, 100, 255, 256, 257, 1000, 1025, 4099, 8191, 8192, 8193, 16385, 50021])
def test_classes(classes):
    rng = np.random.default_rng(classes)
    x = (3 * rng.standard_normal((5, classes))).astype(np.float32)
    tokens = rng.integers(0, classes, 5)
    check(x, tokens, min(5, classes))
    check(x, tokens, 0, pad=3)


@pytest.mark.parametrize("top", [1, 2, 7, 20, 63, 64])
@pytest.mark.parametrize("classes", [64, 777, 20000])
def test_top(top, classes):
    rng = np.random.default_rng(top + classes)
    x = (3 * rng.standard_normal((9, classes))).astype(np.float32)
    check(x, rng.integers(0, classes, 9), top, pad=1)


@pytest.mark.parametrize("classes", [64, 300, 9000, 40000])
def test_equal_logits_go_to_the_lowest_id(classes):
    rng = np.random.default_rng(classes)
    x = np.zeros((6, classes), np.float32)
    x[1] = -0.0
    x[1, ::2] = 0.0
    x[2] = rng.integers(0, 3, classes)
    x[3] = np.arange(classes) // 7
    x[4] = -(np.arange(classes) // 7)
    x[5, -1] = 1
    check(x, np.zeros(6, int), 64)


@pytest.mark.parametrize("ascending", [True, False])
def test_sorted_rows(ascending):
    x = np.linspace(-20, 20, 30000, dtype=np.float32)[None]
    check(x if ascending else x[:, ::-1].copy(), np.array([17]), 50)


def test_padded_places_and_far_tokens():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((4, 50)).astype(np.float32)
    logp, *_ = score(x, np.array([-1, 50, 2 ** 31 - 1, -2 ** 31]), 0)
    np.testing.assert_array_equal(logp, 0)
    np.testing.assert_array_equal(score(x, np.array([-1, 3, 5, 49]), 0, only_logp=True)[0], 0)


def test_masked_logits():
    """-infinity and the type's lowest value add nothing; whole rows of them are defined."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((4, 9000)).astype(np.float32)
    x[0, 10:8999] = -np.inf
    x[1, 1:] = -np.inf
    x[2, 5:] = np.finfo(np.float32).min
    x[3] = np.finfo(np.float32).min
    tokens = np.array([3, 0, 2, 8])
    logp, lse, ent, ids, best = score(x, tokens, 6)
    rp, rl, re, ri, rb = serving.token_logprobs(x, tokens, 6)
    np.testing.assert_array_equal(ids, ri)
    for got, ref in ((logp, rp), (lse, rl), (ent, re), (best, rb)):
        np.testing.assert_allclose(got, ref, rtol=4e-6, atol=4e-6)
    assert ent[1] == 0 and logp[1] == 0


def test_rows_that_are_no_numbers_leave_the_others_alone():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, 10000)).astype(np.float32)
    clean = score(x, np.arange(6), 4)
    x[1] = -np.inf
    x[2, 77] = np.inf
    x[3, 9999] = np.nan
    x[4, 0] = -np.nan
    logp, lse, ent, ids, best = score(x, np.arange(6), 4)
    assert np.isneginf(lse[1]) and np.isnan(lse[2:5]).all() and np.isnan(ent[1:5]).all() and np.isnan(logp[1:5]).all()
    assert np.isnan(best[1:5]).all() and ((ids >= 0) & (ids < 10000)).all()
    np.testing.assert_array_equal(ids[1], np.arange(4))
    for a, b in zip(clean, (logp, lse, ent, ids, best)):
        np.testing.assert_array_equal(a[[0, 5]], b[[0, 5]])


def test_far_rows():
    """Rows past 2^31 elements, a stride of its own."""
    rows, classes, stride = 5, 9000, 600_000_000
    G.say("token_logprobs over rows 2.4 GB apart")
    rng = np.random.default_rng(4)
    x = rng.standard_normal((rows, classes)).astype(np.float32)
    buf = DeviceArray(((rows - 1) * stride + classes,))
    for i in range(rows):
        capi.lib().copy_to_device(buf.ptr + 4 * i * stride, x[i].ctypes.data, 4 * classes)
    logp, tk = DeviceArray((rows,)), ints(np.arange(rows))
    capi.check(capi.lib().token_logprobs(buf.ptr, stride, tk.ptr, rows, classes, logp.ptr, None, None, None, None, 0), "token_logprobs")
    np.testing.assert_array_equal(logp.numpy(), score(x, np.arange(rows), 0)[0])


@pytest.mark.parametrize("classes", [1, 2, 5, 64, 1001, 4096, 4097, 20000])
@pytest.mark.parametrize("pad", [0, 3])
def test_gradient(classes, pad):
    """Each element is p, off by 2 (r + 4) half steps, times d_logp and the entropy's factor."""
    rng = np.random.default_rng(classes)
    x = (3 * rng.standard_normal((6, classes))).astype(np.float32)
    tokens = rng.integers(0, classes, 6)
    tokens[2], tokens[4] = -1, classes
    d_logp, d_ent = rng.standard_normal(6).astype(np.float32), rng.standard_normal(6).astype(np.float32)
    _, rl, re, _, _ = serving.token_logprobs(x, tokens, 1)
    lse, ent = rl.astype(np.float32), re.astype(np.float32)
    r = (np.ptp(x, -1) + np.abs(lse) + 4)[:, None]
    p = np.exp(x.astype(np.float64) - rl[:, None])
    size = np.abs(d_logp)[:, None] + np.abs(d_ent)[:, None] * (np.abs(x - lse[:, None]) + np.abs(ent)[:, None] + 1)
    got = gradient(x, tokens, lse, ent, d_logp, d_ent, pad, 1)
    tol = 4 * U * r * p * size + 2 * U * np.abs(d_logp)[:, None]
    assert (np.abs(got - serving.token_logprobs_bwd(x, tokens, d_logp, d_ent)) <= tol).all()
    zero = np.zeros(6, np.float32)
    assert (np.abs(gradient(x, tokens, lse, None, d_logp, None) - serving.token_logprobs_bwd(x, tokens, d_logp, zero)) <= tol).all()
    assert (np.abs(gradient(x, tokens, lse, ent, None, d_ent) - serving.token_logprobs_bwd(x, tokens, zero, d_ent)) <= tol).all()
    np.testing.assert_array_equal(gradient(x, tokens, lse, ent, d_logp, d_ent, pad, in_place=True), got)


def test_gradient_against_differences():
    """Central differences of the kernel's own forward: the step h leaves h^2 / 6
    of the third derivative (below 1 here) and the roundings of f over h."""
    rng = np.random.default_rng(6)
    x = rng.standard_normal((1, 40)).astype(np.float32)
    tokens, h = np.array([7]), np.float32(2.0 ** -5)
    _, lse, ent, _, _ = score(x, tokens, 0)
    got = gradient(x, tokens, lse, ent, np.ones(1), np.full(1, 0.5))
    for j in range(40):
        up, down = x.copy(), x.copy()
        up[0, j] += h
        down[0, j] -= h
        f = [s[0][0].astype(np.float64) + 0.5 * s[2][0] for s in (score(up, tokens, 0), score(down, tokens, 0))]
        step = np.float64(up[0, j]) - down[0, j]
        assert abs((f[0] - f[1]) / step - got[0, j]) <= h * h / 6 + 16 * 8 * U / h


def test_gradient_of_masked_logits():
    rng = np.random.default_rng(7)
    x = rng.standard_normal((2, 500)).astype(np.float32)
    x[0, 100:] = -np.inf
    x[1, 3:] = np.finfo(np.float32).min
    tokens = np.array([4, 1])
    _, rl, re, _, _ = serving.token_logprobs(x, tokens, 1)
    one = np.ones(2, np.float32)
    got = gradient(x, tokens, rl, re, one, one)
    ref = serving.token_logprobs_bwd(np.where(np.isinf(x), -1e30, x), tokens, one, one)
    np.testing.assert_allclose(got, ref, rtol=0, atol=4e-6)
    assert (got[0, 100:] == 0).all() and (got[1, 3:] == 0).all()


def test_gradient_of_more_rows_than_one_grid_takes():
    """2^24 rows and a few: each block of 4099 rows, alike, gets the same gradient."""
    rng = np.random.default_rng(8)
    rows, classes, block = (1 << 24) + 11, 3, 4099
    x = rng.standard_normal((block, classes)).astype(np.float32)
    tokens = rng.integers(-1, classes, block)
    _, lse, ent, _, _ = serving.token_logprobs(x, tokens, 1)
    d_logp, d_ent = rng.standard_normal(block).astype(np.float32), rng.standard_normal(block).astype(np.float32)
    one = gradient(x, tokens, lse.astype(np.float32), ent.astype(np.float32), d_logp, d_ent)
    many = lambda a: np.resize(a, (rows, *a.shape[1:]))  # noqa: E731
    got = gradient(many(x), many(tokens), many(lse.astype(np.float32)), many(ent.astype(np.float32)), many(d_logp), many(d_ent))
    np.testing.assert_array_equal(got, many(one))


def check_long(x, tokens, top, **more):
    """As check, for threads that take many chunks of 4096 logits (16 of each) in
    turn: n chunks add 16 n roundings and, where the maximum rises, 3 each (the
    factor's exp, two steps, and its product).  Only logits within 104 of the
    maximum count (e^-104 is 0 in fp32)."""
    rows, classes = x.shape
    logp, lse, ent, ids, best = score(x, tokens, top, **more)
    rp, rl, re, ri, rb = serving.token_logprobs(x, tokens, top)
    r = np.minimum(np.where(np.isinf(x), 0, x.max(-1, keepdims=True).astype(np.float64) - x).max(-1), 104)
    off = U * (r + 19 * -(-classes // 4096) + 64 + 2 * np.log2(classes + 1))
    with np.errstate(invalid="ignore"):  # of a logit of -infinity both are
        assert ((logp == rp) | (np.abs(logp - rp) <= off + 2 * U * np.abs(rp))).all()
    assert (np.abs(lse - rl) <= off + 2 * U * (np.abs(rl) + np.abs(x.max(-1)))).all()
    assert (np.abs(ent - re) <= 2 * off * (1 + np.minimum(r, 40))).all()
    if top:
        np.testing.assert_array_equal(ids, ri)
        with np.errstate(invalid="ignore"):
            assert ((best == rb) | (np.abs(best - rb) <= off[:, None] + 2 * U * np.abs(rb))).all()


def rows_of_all_kinds(rng, rows, classes):
    """Rows in turn: normal, rising and falling (every chunk has new alternatives, or
    none), ties that pass the chunks' ends, whole chunks of -infinity (the first, the
    last, all but one), and the largest ones in a late chunk."""
    x = (3 * rng.standard_normal((rows, classes))).astype(np.float32)
    x[1::7].sort(-1)
    x[2::7] = -np.sort(-x[2::7])
    x[3::7] = np.round(x[3::7])
    x[4::7, :4096] = -np.inf
    x[5::7, 4096:] = -np.inf
    x[5::7, -1] = 1
    x[6::7, classes - 700:] += 9
    return x


@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
@pytest.mark.parametrize("rows, classes", [(1100, 9001), (2100, 4097), (1030, 16384), (600, 20001), (700, 12289), (300, 32001)])
def test_rows_of_several_chunks(rows, classes, top):
    """More rows than half of what fills the chip (256 CUs): a workgroup walks a row's
    chunks in turn (the first three), or some of them (two or more pieces a row)."""
    rng = np.random.default_rng(rows + top)
    check_long(rows_of_all_kinds(rng, rows, classes), rng.integers(-1, classes + 1, rows), top, pad=top % 3)


@pytest.mark.parametrize("top", [0, 5, 20, 64])
@pytest.mark.parametrize("rows, classes", [(8, 131072), (3, 151936), (8, 151936), (2, 256000), (1, 262145), (7, 300000), (1, 1100000)])
def test_large_vocabularies(rows, classes, top):
    """Rows in more pieces than a wave has lanes, and than are joined at a time (64)."""
    rng = np.random.default_rng(rows + classes + top)
    check_long(rows_of_all_kinds(rng, rows, classes), rng.integers(0, classes, rows), top)


@pytest.mark.parametrize("rows", [1, 1100])
def test_no_numbers_in_a_late_chunk(rows):
    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, 9001)).astype(np.float32)
    tokens = rng.integers(0, 9001, rows)
    clean = score(x, tokens, 6)
    bad = x.copy()
    bad[0::5, 8999], bad[1::5, 5000] = np.nan, np.inf
    logp, lse, ent, ids, best = score(bad, tokens, 6)
    for n in range(2):
        assert all(np.isnan(a[n::5]).all() for a in (logp, lse, ent, best))
    assert ((ids >= 0) & (ids < 9001)).all()
    others = np.arange(rows) % 5 > 1
    for a, b in zip(clean, (logp, lse, ent, ids, best)):
        np.testing.assert_array_equal(a[others], b[others])


@pytest.mark.parametrize("rows, classes", [(5, 1000), (3, 20000), (1100, 5000)])
def test_lse_in_two_floats(rows, classes):
    """lse + lse_rest has ln s to its own roundings, however far the logits are from
    0; the other outputs are those of token_logprobs, and rows that are no numbers
    have no rest."""
    rng = np.random.default_rng(rows)
    x = (2 * rng.standard_normal((rows, classes)) + 10.0 ** rng.integers(0, 7, (rows, 1))).astype(np.float32)
    x[1], x[2, 3] = -np.inf, np.inf
    G.say(f"token_logprobs_ex rows={rows} classes={classes}")
    dx, tk = DeviceArray.from_numpy(x), ints(np.zeros(rows))
    logp, lse, rest, ent = (DeviceArray((rows,)) for _ in range(4))
    capi.check(capi.lib().token_logprobs_ex(dx.ptr, classes, tk.ptr, rows, classes, logp.ptr, lse.ptr, rest.ptr, ent.ptr, None, None, 0),
               "token_logprobs_ex")
    for a, b in zip((logp, lse, ent), score(x, np.zeros(rows, int), 0)):
        np.testing.assert_array_equal(a.numpy(), b)
    good = np.ones(rows, bool)
    good[1:3] = False
    assert (rest.numpy()[1:3] == 0).all()
    m = x[good].max(-1).astype(np.float64)
    logs = np.log(np.exp(x[good] - m[:, None]).sum(-1))
    got = (lse.numpy()[good].astype(np.float64) - m) + rest.numpy()[good]
    assert (np.abs(got - logs) <= U * (64 + 19 * 2 + np.ptp(x[good], -1) + 4 * logs)).all()
