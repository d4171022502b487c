"""The 4-bit cache through the C ABI against a NumPy oracle: what is written is
right to the bit, at the right slots and nowhere else; what is read back is the
same; attention over it agrees with float64 for one row and many, page ends,
padded batches, rows that see nothing, and slots that hold no numbers."""

import time

import numpy as np
import pytest

import gpu_helpers as G
from ember_amd import capi
from ember_amd.capi import DeviceArray
from oracle import serving
from serving_helpers import Bytes, Pair, ints, table

pytestmark = pytest.mark.gpu


def normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def same_slots(p):
    for name, dev, host in (("codes", p.codes, p.host.codes), ("scales", p.scales, p.host.scales)):
        for d, h in zip(dev, host):
            np.testing.assert_array_equal(d.numpy(), h, err_msg=name)


# ---- writing and reading ----


def hard_rows(D):
    """Rows whose groups are zeros, ties, borders of the scale, and no numbers."""
    rng = np.random.default_rng(5)
    rows = [np.zeros(32), -np.zeros(32), np.linspace(-6, 6, 32), np.linspace(-1, 1, 32) * 1e-30, np.full(32, 1e-45),
            np.array([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5] * 4), -np.array([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5] * 4),
            np.nextafter(np.float32(6), np.float32(7)) * np.linspace(-1, 1, 32), np.full(32, 1.5), np.full(32, -3 * 2.0 ** 90),
            np.linspace(0, 1.99 * 2.0 ** 126, 32), np.linspace(-1, 1, 32) * 2.0 ** -119, np.linspace(-1, 1, 32) * 2.0 ** -122]
    for bad in (np.inf, -np.inf, np.nan, 2.0 ** 127, np.finfo(np.float32).max):
        x = rng.standard_normal(32)
        x[7] = bad
        rows.append(x)
    rows += [rng.standard_normal(32) * 10.0 ** rng.integers(-30, 30) for _ in range(110)]
    x = np.array(rows, np.float32)  # a multiple of 4 groups
    return x[:len(x) // (D // 32) * (D // 32)].reshape(-1, D)


@pytest.mark.parametrize("D", [32, 64, 128])
def test_write_rounds_as_the_format_says(D):
    x = hard_rows(D)
    T = len(x)
    p = Pair((T + 15) // 16, 1, 16, D, [np.arange((T + 15) // 16)])
    p.write(x[None, :, None], -x[None, ::-1, None])
    same_slots(p)
    k, v = p.read(T)
    for got, ref in zip((k, v), p.host.read(T)):
        np.testing.assert_array_equal(got, ref.astype(np.float32))


@pytest.mark.parametrize("B, T, H, D, page, start, count", [
    (1, 1, 1, 32, 16, None, None),
    (3, 5, 2, 64, 16, [0, 14, 31], None),            # across page ends
    (4, 7, 5, 128, 32, [3, 0, 57, 20], [7, 0, 4, 9]),  # none valid, some valid, a count past T
    (2, 33, 3, 32, 64, [0, 40], [33, 20]),
    (3, 4, 1, 64, 16, [-2, 62, 1000], None),         # before the sequence, past its table
    (2, 600, 16, 128, 256, [1, 100], [600, 411]),
])
def test_write_and_read_slots(B, T, H, D, page, start, count):
    rng = np.random.default_rng(B * T + D)
    places = -(-(max(start or [0]) + T) // page) if max(start or [0]) < 900 else 64 // page
    tab, pages = table(rng, B, places)
    p = Pair(pages, H, page, D, tab, fill=0x5A)
    got, ref = p.write(normal(rng, B, T, H, D), normal(rng, B, T, H, D), start, count, stride_pad=4)
    np.testing.assert_array_equal(got, ref)
    same_slots(p)
    for got, ref in zip(p.read(T, start, count), p.host.read(T, start, count)):
        np.testing.assert_array_equal(got, ref.astype(np.float32))


@pytest.mark.parametrize("D", [32, 64, 128])
def test_a_large_context_read_back(D):
    """Over 192 MiB of values at once, as the same tokens read in parts."""
    rng = np.random.default_rng(D)
    H, T = 1024 // D, 25000
    p = filled(rng, 1, H, 256, D, 600)
    p.table = ints(np.tile(p.host.table, (1, 33)))   # the same tokens over and over
    p.view.page_table, p.view.max_pages = p.table.ptr, 33 * p.host.table.shape[1]
    p.host.table = np.tile(p.host.table, (1, 33))
    k, v = p.read(T, count=[T - 7])
    assert k.nbytes + v.nbytes > 192 << 20
    for t0 in (0, 9000, 24500):
        pk, pv = p.read(500, start=[t0], count=[min(500, T - 7 - t0)])
        np.testing.assert_array_equal(k[:, t0:t0 + 500], pk)
        np.testing.assert_array_equal(v[:, t0:t0 + 500], pv)


@pytest.mark.parametrize("fault", [-1, 7, 2 ** 31 - 1, -2 ** 31])
def test_pages_that_are_not_there(fault):
    """Tokens of a page outside the cache are dropped, read as zero and not seen."""
    rng = np.random.default_rng(11)
    tab = np.array([[0, fault, 2], [3, 4, fault]], np.int32)
    p = Pair(7, 2, 16, 64, tab)
    k, v = normal(rng, 2, 48, 2, 64), normal(rng, 2, 48, 2, 64)
    p.write(k, v)
    same_slots(p)
    for got, ref in zip(p.read(48), p.host.read(48)):
        np.testing.assert_array_equal(got, ref.astype(np.float32))
    p.check_attention(normal(rng, 2, 3, 4, 64), True, start=[45, 20])
    p.check_attention(normal(rng, 2, 1, 4, 64), True, start=[17, 47])


def test_next_without_rows_and_no_next():
    p = Pair(2, 1, 16, 32, [[0], [1]])
    start, nxt = ints([3, 9]), ints([-1, -1])
    p.write(np.ones((2, 1, 1, 32), np.float32), np.ones((2, 1, 1, 32), np.float32), [3, 9])
    G.say("kv_cache_write of no rows")
    capi.check(capi.lib().kv_cache_write(p.view, None, None, 0, 0, 0, 0, start.ptr, None, nxt.ptr), "kv_cache_write")
    np.testing.assert_array_equal(nxt.numpy(), [3, 9])
    same_slots(p)


# ---- attention ----


def filled(rng, B, H, page, D, L, fill=255):
    """A cache of B sequences with L tokens each (slots past them hold `fill`)."""
    tab, pages = table(rng, B, -(-L // page))
    p = Pair(pages, H, page, D, tab, fill)
    p.write(normal(rng, B, L, H, D), normal(rng, B, L, H, D))
    return p


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("L", [1, 2, 15, 16, 17, 31, 33, 64, 127, 200])
def test_one_token(D, L):
    rng = np.random.default_rng(L + D)
    p = filled(rng, 2, 2, 16, D, L)
    p.check_attention(normal(rng, 2, 1, 4, D), True, start=[L - 1, (L - 1) // 2])


@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 9, 16, 17])
@pytest.mark.parametrize("T", [1, 3, 8])
def test_groups_of_heads(group, T):
    rng = np.random.default_rng(group * T)
    p = filled(rng, 2, 3, 32, 64, 90)
    p.check_attention(normal(rng, 2, T, 3 * group, 64), True, start=[90 - T, 7])


@pytest.mark.parametrize("D, T, G_, L, causal", [
    (128, 40, 4, 150, True), (64, 33, 1, 97, True), (32, 70, 2, 130, True), (128, 64, 1, 64, True), (64, 129, 3, 200, False),
    (32, 5, 1, 300, False), (128, 17, 8, 80, False),
])
def test_many_rows(D, T, G_, L, causal):
    rng = np.random.default_rng(D + T)
    p = filled(rng, 2, 2, 16, D, L)
    p.check_attention(normal(rng, 2, T, 2 * G_, D), causal, start=[L - T, (L - T) // 3])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("T", [4, 50])
def test_padded_batch_and_empty_rows(causal, T):
    """Counts below T, sequences with nothing in them, rows before the start."""
    rng = np.random.default_rng(T)
    p = filled(rng, 5, 2, 16, 64, 80)
    o, lse = p.check_attention(normal(rng, 5, T, 6, 64), causal, start=[80 - T, 3, 0, 0, -2], count=[T, 2, 0, 1, T - 1])
    assert (o[2] == 0).all() and np.isneginf(lse[2]).all()
    assert (o[1, 2:] == 0).all() and np.isneginf(lse[1, :, 2:]).all()
    if causal:
        assert (o[4, :2] == 0).all() and np.isneginf(lse[4, :, :2]).all()


@pytest.mark.parametrize("T", [1, 6, 40])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_what_is_no_number_reaches_only_who_sees_it(T, D):
    """NaN keys and values late in a sequence: rows before them stay finite."""
    rng = np.random.default_rng(T + D)
    L = 70
    tab, pages = table(rng, 2, 5)
    p = Pair(pages, 2, 16, D, tab)
    k, v = normal(rng, 2, L, 2, D), normal(rng, 2, L, 2, D)
    v[0, L - 1, 0, D - 1] = np.nan
    v[1, L - T // 2 - 1, 1, 0] = np.inf
    k[1, L - 1, 0, 3] = np.nan
    p.write(k, v)
    q = normal(rng, 2, T, 4, D)
    o, _ = p.check_attention(q, True, start=[L - T, L - T])
    assert np.isnan(o[0, -1, 0, D - 32:]).all() and np.isfinite(o[0, -1, 0, :D - 32]).all()
    if T > 1:
        assert np.isfinite(o[0, :-1]).all()
    p.check_attention(q, True, start=[L - T - 10, 5])


def test_long_sequence_and_splits():
    """Keys split over workgroups, and joined: 5000 tokens of one sequence."""
    rng = np.random.default_rng(3)
    p = filled(rng, 1, 1, 256, 32, 5000)
    p.check_attention(normal(rng, 1, 1, 2, 32), True, start=[4999])
    p.check_attention(normal(rng, 1, 2, 1, 32), True, start=[130])


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("T", [20, 70])
def test_many_rows_and_splits(D, T):
    """Many rows with their keys split over workgroups, sequences of very different lengths."""
    rng = np.random.default_rng(D * T)
    p = filled(rng, 3, 1, 64, D, 1700)
    p.check_attention(normal(rng, 3, T, 2, D), True, start=[1700 - T, 600, 0], count=[T, T, 3])
    p.check_attention(normal(rng, 3, T, 2, D), False, start=[1700 - T, 600, 0], count=[T, 5, T])


@pytest.mark.parametrize("B", [65, 150, 1100])
@pytest.mark.parametrize("T, G_", [(1, 1), (1, 3), (2, 4), (9, 5)])
def test_many_sequences(B, T, G_):
    """More sequences than a wave has lanes, and more than are planned for, of all lengths."""
    rng = np.random.default_rng(B + T)
    tab, pages = table(rng, B, 3)
    p = Pair(pages, 1, 16, 32, tab)
    p.write(normal(rng, B, 48, 1, 32), normal(rng, B, 48, 1, 32))
    start = rng.integers(-1, 48 - T + 1, B)
    p.check_attention(normal(rng, B, T, G_, 32), True, start=start, count=rng.integers(0, T + 1, B))


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("T, G_", [(1, 1), (2, 1), (1, 2), (1, 3), (3, 1), (1, 4), (2, 2), (5, 1), (1, 8), (4, 5)])
def test_few_rows_and_splits(D, T, G_):
    """Two, four and eight rows to a workgroup, with keys cut into pieces (of 640 at
    least): lengths, counts, NaN in one piece and pages that are not there."""
    rng = np.random.default_rng(D * T + G_)
    L, page = 1900, 64
    tab, pages = table(rng, 4, 30)
    p = Pair(pages, 2, page, D, tab)
    k, v = normal(rng, 4, L, 2, D), normal(rng, 4, L, 2, D)
    v[0, 1400, 1, D - 1] = np.nan
    k[0, L - 1, 0, 3] = np.inf
    p.write(k, v, count=[L, 900, 500, L])
    p.host.table[3, 12:23] = -1
    p.table = ints(p.host.table)
    p.view.page_table = p.table.ptr
    q = normal(rng, 4, T, 2 * G_, D)
    start = [L - T, 900 - T, 40, L - T - 11]
    o, _ = p.check_attention(q, True, start=start)
    assert np.isnan(o[0, :, G_:, D - 32:]).all() and np.isfinite(o[1:]).all()
    p.check_attention(q, False, start=start, count=[T, 1, 0, T])


def test_sequences_of_very_different_lengths():
    """One long sequence among many short and empty ones, cut into pieces."""
    rng = np.random.default_rng(20)
    B, lengths = 70, np.zeros(70, int)
    lengths[[3, 66]] = 3000, 900
    lengths[10:60] = rng.integers(0, 40, 50)
    tab = np.full((B, 12), -1, np.int32)
    need, n = -(-lengths // 256), 0
    for b in range(B):
        tab[b, :need[b]] = np.arange(n, n + need[b])
        n += need[b]
    p = Pair(n, 1, 256, 64, tab)
    for b in np.nonzero(lengths)[0]:
        k, v = np.zeros((2, B, lengths[b], 1, 64), np.float32)
        k[b], v[b] = normal(rng, lengths[b], 1, 64), normal(rng, lengths[b], 1, 64)
        p.write(k, v, count=np.where(np.arange(B) == b, lengths[b], 0))
    for T, heads in ((1, 2), (2, 3), (30, 2)):
        p.check_attention(normal(rng, B, T, heads, 64), True, start=lengths - T)


@pytest.mark.parametrize("T, G_, heads", [(1, 1, 32), (3, 1, 32), (5, 1, 16), (24, 1, 6)])
def test_long_sequences_among_units_of_several_rounds(T, G_, heads):
    """More units than the chip takes in four rounds: the long sequences are cut all the same."""
    rng = np.random.default_rng(T)
    B, page, D = 70, 64, 128
    lengths = rng.integers(0, 40, B)
    lengths[[2, 68]] = 2500, 1400
    need, n = -(-lengths // page), 0
    tab = np.full((B, need.max()), -1, np.int32)
    for b in range(B):
        tab[b, :need[b]] = np.arange(n, n + need[b])
        n += need[b]
    p = Pair(n, heads, page, D, tab)
    for a, b in zip((*p.host.codes, *p.host.scales), (*p.codes, *p.scales)):
        a[...] = rng.integers(120, 126, a.shape) if a is p.host.scales[0] or a is p.host.scales[1] else rng.integers(0, 256, a.shape)
        b.dev = Bytes(a).dev
    p.view.k_codes, p.view.v_codes, p.view.k_scales, p.view.v_scales = (x.ptr for x in (*p.codes, *p.scales))
    o, lse = p.check_attention(normal(rng, B, T, heads * G_, D), True, start=lengths - T)


def test_a_long_sequence_does_not_decide():
    """One of 32768 tokens among 79 of 500 takes less than 80 of 2000, twice as many tokens in all."""
    B, heads, page, D = 80, 32, 256, 128
    p = Pair(8, heads, page, D, np.arange(128)[None].repeat(B, 0) % 8, fill=0x77)
    q, o = (DeviceArray.from_numpy(np.ones((B, 1, heads, D), np.float32)) for _ in range(2))

    def seconds(lengths):
        start = ints(np.array(lengths) - 1)
        st = (heads * D, D, heads * D)
        best = np.inf
        for _ in range(5):
            start.numpy()  # waits
            t0 = time.perf_counter()
            for _ in range(20):
                rc = capi.lib().kv_cache_attention(p.view, q.ptr, o.ptr, None, 1, heads, G.scale_for(D), 1, *st, *st, start.ptr, None)
                capi.check(rc, "kv_cache_attention")
            start.numpy()  # waits
            best = min(best, time.perf_counter() - t0)
        return best

    G.say("kv_cache_attention B=80 heads=32 D=128, 32768 and 79 x 500, and 80 x 2000")
    assert seconds([32768] + 79 * [500]) < seconds(80 * [2000])


@pytest.mark.parametrize("pages, places", [(0, 2), (3, 0), (0, 0)])
def test_caches_of_nothing(pages, places):
    """No pages, or no place for any: nothing is written, read or seen."""
    rng = np.random.default_rng(21)
    p = Pair(pages, 2, 16, 64, np.zeros((2, places), np.int32))
    got, ref = p.write(normal(rng, 2, 5, 2, 64), normal(rng, 2, 5, 2, 64))
    np.testing.assert_array_equal(got, ref)
    for x in p.read(5):
        assert (x == 0).all()
    for T in (1, 5, 50):
        o, lse = p.attention(normal(rng, 2, T, 4, 64), True)
        assert (o == 0).all() and np.isneginf(lse).all()


def test_scores_of_all_sizes():
    """Scores from -300 to 300, growing along the keys (the maximum is raised often), and scale 0."""
    rng = np.random.default_rng(8)
    tab, pages = table(rng, 1, 10)
    p = Pair(pages, 1, 16, 64, tab)
    k = normal(rng, 1, 160, 1, 64) * np.linspace(0.01, 40, 160, dtype=np.float32)[None, :, None, None]
    p.write(k, normal(rng, 1, 160, 1, 64))
    q = normal(rng, 1, 5, 4, 64)
    o, lse = p.attention(q, True, start=[155])
    ro, rl, weight, reach = p.host.attention(q, True, G.scale_for(64), [155], None)
    off = 2 * 2.0 ** -24 * (64 + 8) * reach.transpose(0, 2, 1)[..., None]
    assert (np.abs(o - ro) <= (2 * off + 2.0 ** -23 * 176) * weight).all()
    p.check_attention(q, True, scale=0.0, start=[155])


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("T", [1, 3, 7, 50, 140])
@pytest.mark.parametrize("size", [1e5, 1e7, 1e9, 1e12, 1e20])
def test_large_scores(size, T, D):
    """Scores of `size` times 1, 1.5, 2, 3, ... 12, 16 keys of each, some rows' all
    negative.  A row's largest are equal to the bit (keys alike) and all others
    further below than the scores' roundings reach, 2 (D + 8) half steps of 12
    sizes and less than 0.01 of `size`: o is the mean of the largest ones' values,
    off by the roundings of its sum."""
    rng = np.random.default_rng(D + T)
    L, q_heads = 128, 1
    tab, pages = table(rng, 2, 8)
    p = Pair(pages, 1, 16, D, tab)
    level = np.array([1, 1.5, 2, 3, 4, 6, 8, 12], np.float32).repeat(16)
    k = np.broadcast_to(level[None, :, None, None], (2, L, 1, D)).copy()
    p.write(k, normal(rng, 2, L, 1, D))
    q = size / (D * G.scale_for(D)) * rng.uniform(0.5, 1.5, (2, T, q_heads, D))
    q[:, 1::2] *= -1
    q = q.astype(np.float32)
    start = [max(L - T, 0), 0]
    o, lse = p.attention(q, True, start=start)
    ro, rl, weight, reach = p.host.attention(q, True, G.scale_for(D), start, None)
    assert (np.abs(o - ro) <= 2 * 2.0 ** -24 * (L + 16) * weight).all()
    assert (np.abs(lse - rl) <= 2.0 ** -23 * ((D + 8) * reach + np.abs(rl) + 16)).all()


@pytest.mark.parametrize("T", [1, 3, 7, 50, 140])
@pytest.mark.parametrize("scale", [1e-40, 1e-30, 0.7, 1.3 * 2.0 ** 100, 1e38])
def test_scales_of_all_sizes(scale, T):
    """A scale and queries whose product is of ordinary size, to the ends of fp32's range."""
    rng = np.random.default_rng(T)
    scale = float(np.float32(scale))
    p = filled(rng, 1, 1, 16, 64, 150)
    q = (normal(rng, 1, T, 1, 64) * min(0.125 / scale, 2.0 ** 120)).astype(np.float32)
    p.check_attention(q, True, scale=scale, start=[150 - T])


@pytest.mark.parametrize("T", [1, 3, 7, 50, 140])
@pytest.mark.parametrize("sizes", [(-100, 100), (100, -100), (120, -115), (-140, 20), (20, -60)])
def test_queries_and_keys_of_all_sizes(sizes, T):
    """Queries about 2^a, other rows up to 2^40 smaller, and keys about 2^b, under a
    scale that makes scores of ordinary size."""
    rng = np.random.default_rng(T)
    a, b = sizes
    tab, pages = table(rng, 1, 10)
    p = Pair(pages, 1, 16, 64, tab)
    p.write(normal(rng, 1, 150, 1, 64) * np.float32(2.0 ** b), normal(rng, 1, 150, 1, 64))
    apart = 2.0 ** -rng.integers(0, 41, (1, T, 2, 1))
    apart[0, 0] = 1
    q = (normal(rng, 1, T, 2, 64) * apart * 2.0 ** a).astype(np.float32)
    p.check_attention(q, True, scale=float(np.float32(0.1 * 2.0 ** -(a + b))), start=[150 - T])


@pytest.mark.parametrize("T", [1, 3, 7, 50, 140])
def test_scale_zero_whatever_the_products(T):
    """Products of 10^37 with a scale of 0: every key that a row sees weighs the same."""
    rng = np.random.default_rng(T)
    tab, pages = table(rng, 1, 10)
    p = Pair(pages, 1, 16, 64, tab)
    p.write(normal(rng, 1, 160, 1, 64) * np.float32(2.0 ** 60), normal(rng, 1, 160, 1, 64))
    p.check_attention(normal(rng, 1, T, 1, 64) * np.float32(2.0 ** 60), True, scale=0.0, start=[160 - T])


@pytest.mark.parametrize("first", [0, -17, -19, -40, 17, 19, 40])
@pytest.mark.parametrize("D, T", [(32, 21), (64, 50), (128, 50)])
def test_many_rows_over_scales_far_apart(D, T, first):
    """Tokens and groups of very different sizes: the first token's keys and values
    are about 2^first times the others'."""
    rng = np.random.default_rng(D + first + 40)
    L = 200
    tab, pages = table(rng, 2, 13)
    p = Pair(pages, 2, 16, D, tab)
    sizes = lambda spread: 2.0 ** rng.integers(-spread, spread + 1, (2, L, 2, D // 32)).repeat(32, -1)  # noqa: E731
    groups = 2.0 ** rng.integers(-5, 6, D // 32).repeat(32)
    k, v = normal(rng, 2, L, 2, D) / groups, normal(rng, 2, L, 2, D) * sizes(6)
    k *= 2.0 ** np.minimum(-first, 0)
    k[:, 0] *= 2.0 ** first
    v[:, 0] *= 2.0 ** first
    k[1, 5:20] = 0
    v[1, 60:70] = -0.0
    p.write(k.astype(np.float32), v.astype(np.float32))
    p.check_attention((normal(rng, 2, T, 6, D) * groups).astype(np.float32), True, start=[L - T, 60])


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("T", [50, 140])
@pytest.mark.parametrize("odd", ["large values", "small values", "small keys", "no number", "no key", "all"])
def test_many_rows_with_one_piece_far_apart(odd, T, D):
    """Keys cut into pieces (of 512 at least), one of which holds what fp16 cannot in
    its first token's units: done again in bf16, and joined with those that were not."""
    rng = np.random.default_rng(D + T)
    L = 2300
    tab, pages = table(rng, 2, 36)
    p = Pair(pages, 1, 64, D, tab)
    k, v = normal(rng, 2, L, 1, D), normal(rng, 2, L, 1, D)
    if odd in ("large values", "all"):
        v[:, 1300:1310] *= np.float32(2.0 ** 18)
    if odd in ("small values", "all"):
        v[:, 1320:1400] *= np.float32(2.0 ** -25)
    if odd in ("small keys", "all"):
        k[:, 1350:1420] *= np.float32(2.0 ** -30)
    if odd in ("no number", "all"):
        v[0, 1290, 0, 5] = np.nan
    if odd in ("no key", "all"):
        k[1, L - 30, 0, 7] = np.inf
    p.write(k, v)
    q = normal(rng, 2, T, 1, D)
    o, lse = p.check_attention(q, True, start=[L - T, L - T])
    assert np.isnan(lse[1, :, -30:]).all() == (odd in ("no key", "all")) and np.isfinite(lse[1, :, :-30]).all()
    p.check_attention(q, True, start=[700, 1380 - T], count=[T, T])


@pytest.mark.parametrize("D, T", [(32, 15), (64, 15), (128, 40), (64, 60)])
def test_many_rows_over_scores_of_all_sizes(D, T):
    """test_scores_of_all_sizes for more than 40 rows, and with pieces.  Weights there
    are two fp16 parts in a unit of 2^-7 of the largest, whose last step is 2^-24:
    each is off by 2^-25 * 2^-7 of the largest at most, where that is more than its
    roundings (columns in which the keys of large weights hold zeros)."""
    rng = np.random.default_rng(T)
    for L in (160, 1300):
        tab, pages = table(rng, 1, -(-L // 16))
        p = Pair(pages, 1, 16, D, tab)
        k = normal(rng, 1, L, 1, D) * np.linspace(0.01, 40, L, dtype=np.float32)[None, :, None, None]
        p.write(k, normal(rng, 1, L, 1, D))
        q = normal(rng, 1, T, 4, D)
        o, lse = p.attention(q, True, start=[L - T])
        ro, rl, weight, reach = p.host.attention(q, True, G.scale_for(D), [L - T], None)
        off = 2 * 2.0 ** -24 * (D + 8) * reach
        floor = 2.0 ** -32 * np.abs(p.host.read(L)[1]).sum(1)[:, None]
        assert (np.abs(o - ro) <= (2 * off.transpose(0, 2, 1)[..., None] + 2.0 ** -23 * (L + 16)) * weight + floor).all()
        assert (np.abs(lse - rl) <= off + 2.0 ** -23 * (np.abs(rl) + L + 16)).all()


@pytest.mark.parametrize("D, T", [(64, 50), (128, 140)])
@pytest.mark.parametrize("less", [0, 6, 11, 13, 14, 17, 19, 24])
def test_many_rows_over_values_below_the_first(D, T, less):
    """Columns in which only the first token has none, and the others' are 2^-less
    of its size elsewhere; few keys and flat weights, so that the bound is near the
    roundings' own size."""
    rng = np.random.default_rng(less)
    L = 5
    tab, pages = table(rng, 1, 1)
    p = Pair(pages, 1, 16, D, tab)
    k, v = normal(rng, 1, L, 1, D) * np.float32(0.01), normal(rng, 1, L, 1, D) * np.float32(2.0 ** (20 - less))
    v[0, 0, 0] = 0
    v[0, 0, 0, :32] = 2.0 ** 20
    p.write(k, v)
    p.check_attention(normal(rng, 1, T, 1, D), False, start=[0], count=[L])


def test_a_row_of_q_that_is_no_number():
    rng = np.random.default_rng(9)
    p = filled(rng, 1, 1, 16, 64, 40)
    q = normal(rng, 1, 3, 2, 64)
    q[0, 1, 0, 5] = np.inf
    q[0, 2, 1, 7] = np.nan
    o, lse = p.attention(q, True, start=[37])
    assert np.isnan(o[0, 1, 0]).all() and np.isnan(o[0, 2, 1]).all() and np.isnan(lse[0, 0, 1]) and np.isnan(lse[0, 1, 2])
    fine = np.isfinite(q).all(-1)
    ro = p.host.attention(np.where(fine[..., None], q, 0), True, G.scale_for(64), [37], None)[0]
    np.testing.assert_allclose(o[fine], ro[fine], rtol=0, atol=2e-5)


def test_small_and_large_sizes_of_numbers():
    """Queries near the ends of fp32's range meet keys near the others."""
    rng = np.random.default_rng(10)
    tab, pages = table(rng, 1, 2)
    p = Pair(pages, 1, 16, 32, tab)
    k = normal(rng, 1, 20, 1, 32) * np.float32(2.0 ** -60)
    p.write(k, normal(rng, 1, 20, 1, 32) * np.float32(2.0 ** 100))
    p.check_attention(normal(rng, 1, 2, 1, 32) * np.float32(2.0 ** 60), True, start=[18])


def test_layouts_and_no_lse():
    rng = np.random.default_rng(12)
    p = filled(rng, 2, 2, 32, 128, 50)
    q = normal(rng, 2, 9, 4, 128)
    o1, _ = p.check_attention(q, True, start=[41, 20])
    o2, _ = p.check_attention(q, True, start=[41, 20], head_major=True)
    o3, none = p.check_attention(q, True, start=[41, 20], want_lse=False)
    assert none is None
    np.testing.assert_array_equal(o1, o2)
    np.testing.assert_array_equal(o1, o3)


def test_shared_pages():
    """Two sequences whose first pages are the same ones."""
    rng = np.random.default_rng(13)
    p = Pair(4, 1, 16, 64, [[0, 1, 2], [0, 1, 3]])
    k, v = normal(rng, 1, 32, 1, 64), normal(rng, 1, 32, 1, 64)
    both = lambda x: np.concatenate([x, np.zeros_like(x)])  # noqa: E731
    p.write(both(k), both(v), count=[32, 0])
    p.write(normal(rng, 2, 5, 1, 64), normal(rng, 2, 5, 1, 64), start=[32, 32])
    p.check_attention(normal(rng, 2, 5, 2, 64), True, start=[32, 32])


def test_calls_repeat_to_the_bit():
    rng = np.random.default_rng(14)
    p = filled(rng, 3, 4, 64, 128, 700)
    q = normal(rng, 3, 1, 16, 128)
    first = p.attention(q, True, start=[699, 300, 64])
    for _ in range(3):
        again = p.attention(q, True, start=[699, 300, 64])
        for a, b in zip(first, again):
            np.testing.assert_array_equal(a, b)


def test_far_slots():
    """Pages whose codes lie past 2^32 bytes from the first."""
    pages, heads, page, D = 70000, 2, 512, 128   # 64 bytes a row: 4.6 GB of codes each
    G.say("kv cache of 70000 pages")
    per = heads * page * D // 2
    codes = [capi.DeviceArray((pages * per // 4,)) for _ in range(2)]
    scales = [capi.DeviceArray((pages * per // 64,)) for _ in range(2)]
    rng = np.random.default_rng(15)
    tab = Bytes(np.array([[pages - 1, 3]], np.int32))
    near = Pair(2, heads, page, D, [[0, 1]])
    far = capi.KVCacheView(codes[0].ptr, scales[0].ptr, codes[1].ptr, scales[1].ptr, tab.ptr, pages, heads, page, D, 1, 2)
    k, v, q = normal(rng, 1, 600, heads, D), normal(rng, 1, 600, heads, D), normal(rng, 1, 1, 4, D)
    near.write(k, v)
    want = near.attention(q, True, start=[599])
    near.view = far
    near.write(k, v)
    for a, b in zip(want, near.attention(q, True, start=[599])):
        np.testing.assert_array_equal(a, b)
    for a, b in zip(near.read(600), near.host.read(600)):
        np.testing.assert_array_equal(a, b.astype(np.float32))


def test_written_step_by_step_as_at_once():
    """A prompt, then tokens one by one: the same cache and, row for row, the same attention as in one call."""
    rng = np.random.default_rng(16)
    B, L, H, D = 2, 45, 2, 64
    k, v, q = (normal(rng, B, L, H, D) for _ in range(3))
    tab, pages = table(rng, B, 3)
    whole = Pair(pages, H, 16, D, tab)
    whole.write(k, v)
    o, lse = whole.check_attention(q, True)
    steps = Pair(pages, H, 16, D, tab)
    at = np.zeros(B, np.int32)
    for t0, t1 in [(0, 30), *[(t, t + 1) for t in range(30, L)]]:
        nxt, _ = steps.write(k[:, t0:t1], v[:, t0:t1], start=at)
        so, sl = steps.attention(q[:, t0:t1], True, start=at)
        np.testing.assert_allclose(so, o[:, t0:t1], rtol=0, atol=4e-6)
        np.testing.assert_allclose(sl, lse[:, :, t0:t1], rtol=0, atol=4e-6)
        at = nxt
    np.testing.assert_array_equal(at, [L, L])
    for a, b in zip((*whole.codes, *whole.scales), (*steps.codes, *steps.scales)):
        np.testing.assert_array_equal(a.numpy(), b.numpy())


def test_oracle_values_agree_with_what_is_read():
    rng = np.random.default_rng(17)
    x = normal(rng, 4, 128)
    codes, scales = serving.quantise(x)
    back = serving.values(codes, scales)
    # Half a step of the grid: at most 1 of 6 in the top half of a group, 1/6 of amax.
    amax = np.abs(x).reshape(4, 4, 32).max(-1)
    assert (np.abs(back - x).reshape(4, 4, 32) <= amax[..., None] / 3).all()
