"""Where the kernels of 8-bit products read (ember_amd/csrc/linear8_shape.h), at the
largest matrices.  CPU only."""

import ctypes as C
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ember_amd", "csrc")
SOURCE = """
#include "linear8_shape.h"
extern "C" unsigned buffer_bytes() { return ember::kBufferBytes; }
extern "C" unsigned lane_offset(unsigned in_tile, int there) { return ember::lane_offset(in_tile, there != 0); }
"""


@pytest.fixture(scope="module")
def shape(tmp_path_factory):
    d = tmp_path_factory.mktemp("linear8_shape")
    (d / "s.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-I", CSRC, "s.cpp", "-o", "s.so"], cwd=d, check=True)
    L = C.CDLL(str(d / "s.so"))
    L.buffer_bytes.restype = L.lane_offset.restype = C.c_uint
    L.lane_offset.argtypes = [C.c_uint, C.c_int]
    return L


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
