"""Where the kernels of 8-bit products read, at the largest matrices, and which of them
a call takes, on a whole card and on parts of one (ember_amd/csrc/linear8_shape.h).
CPU only."""

import ctypes as C
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ember_amd", "csrc")
SOURCE = """
#include "linear8_shape.h"
extern "C" unsigned buffer_bytes() { return ember::kBufferBytes; }
extern "C" unsigned lane_offset(unsigned in_tile, int there) { return ember::lane_offset(in_tile, there != 0); }
extern "C" int few_columns(int64_t n, int64_t m, int gated, int cus) { return ember::few_columns(n, m, gated != 0, cus); }
extern "C" int four_waves(int64_t m, int groups, int cus) { return ember::four_waves(m, groups, cus); }
extern "C" void choose(int64_t n, int64_t m, int groups, int gated, int cus, int *out)
{
    const ember::Choice c = ember::choose(n, m, groups, gated != 0, cus);
    out[0] = c.kernel, out[1] = c.splits, out[2] = c.chunk;
}
extern "C" void without_scratch(int groups, int gated, int *out)
{
    const ember::Choice c = ember::without_scratch(groups, gated != 0);
    out[0] = c.kernel, out[1] = c.splits, out[2] = c.chunk;
}
"""
FEW, SMALL, MID, LARGE = range(4)


@pytest.fixture(scope="module")
def shape(tmp_path_factory):
    d = tmp_path_factory.mktemp("linear8_shape")
    (d / "s.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-I", CSRC, "s.cpp", "-o", "s.so"], cwd=d, check=True)
    L = C.CDLL(str(d / "s.so"))
    L.buffer_bytes.restype = L.lane_offset.restype = C.c_uint
    L.lane_offset.argtypes = [C.c_uint, C.c_int]
    L.few_columns.argtypes = [C.c_int64, C.c_int64, C.c_int, C.c_int]
    L.four_waves.argtypes = [C.c_int64, C.c_int, C.c_int]
    L.without_scratch.argtypes = [C.c_int, C.c_int, C.c_void_p]
    L.choose.argtypes = [C.c_int64, C.c_int64, C.c_int, C.c_int, C.c_int, C.c_void_p]
    return L


def choose(L, *args):
    out = (C.c_int * 3)()
    L.choose(*args, out)
    return tuple(out)


@pytest.mark.parametrize("pitch", [128, 4096, 2 ** 23 - 128, 2 ** 23])
def test_loads_stay_in_the_tile_or_read_nothing(shape, pitch):
    """The lane's share alone is past the buffer where nothing is to be read: a bound that
    leaves out what all lanes share, or that wraps below it, holds as well."""
    size = shape.buffer_bytes()
    for row in (0, 1, 63, 255):  # of a tile's at most 256
        for unit in (0, 16, 48, 64, 112):  # of a row's 128 bytes of a group
            place = row * pitch + unit
            assert shape.lane_offset(place, 1) == place and place + (pitch - 128) + 16 <= size
            past = shape.lane_offset(place, 0)
            assert past >= size and past + 64 + 16 < 2 ** 32  # the kernel for few rows adds up to 64


@pytest.mark.parametrize("gated", [0, 1])
@pytest.mark.parametrize("cus", [32, 64, 128, 256])
def test_choices_cover_k(shape, cus, gated):
    for n in (1, 17, 64, 65, 300, 1025, 8192, 2 ** 20):
        for m in (1, 40, 129, 1000, 4096, 11000, 2 ** 19):
            for groups in (1, 2, 3, 7, 8, 9, 32, 33, 200, 65536):
                kernel, splits, chunk = choose(shape, n, m, groups, gated, cus)
                assert kernel in ((FEW, SMALL, MID, LARGE) if gated else (FEW, SMALL, LARGE))
                assert 1 <= splits <= 16 and (splits - 1) * chunk < groups <= splits * chunk
                if splits > 1:  # scales are read in fours; parts of at most 500 MB
                    assert kernel == SMALL and chunk % 4 == 0 and splits * 4 * (1 + gated) * n * m <= 5e8


def test_rules_follow_the_cards_units(shape):
    """A part of a card with 1/8 of the CUs decides on 1/8 of the columns as the whole one does."""
    for m in (64, 512, 1272, 1280, 2000, 4096, 4100, 5088, 5096, 8160, 8192, 10176, 10240, 16384, 50000):
        for n in (1, 8, 9, 33, 64):
            for gated in (0, 1):
                assert shape.few_columns(n, m * 8, gated, 256) == shape.few_columns(n, m, gated, 32) or m % 64
        for groups in (1, 8, 9, 100):
            assert shape.four_waves(m * 8, groups, 256) == shape.four_waves(m, groups, 32) or m % 16
    assert [shape.four_waves(m, 9, 256) for m in (1, 4096, 4097)] == [1, 1, 0] and not shape.four_waves(1, 8, 256)
    assert [shape.few_columns(9, m, 0, 256) for m in (159 * 32, 159 * 32 + 1, 159 * 64, 159 * 64 + 1)] == [1, 2, 2, 4]
    assert [shape.few_columns(33, m, 1, 256) for m in (255 * 32, 255 * 32 + 1)] == [1, 2]


@pytest.mark.parametrize("groups", [1, 32, 65536])
def test_without_memory_for_sums_there_are_none(shape, groups):
    """Kernels that write to the output: of a product any with one split, of a gated layer the gated tiles."""
    for gated, kernel in ((0, SMALL), (1, MID)):
        out = (C.c_int * 3)()
        shape.without_scratch(groups, gated, out)
        assert tuple(out) == (kernel, 1, groups)
