"""The rules of dma_route.hpp, compiled for the CPU: tiles, parts of k and rows
apart of the products on the DMA tiles.

* every product has a finite estimate, also of fewer than four steps of k, and is
  not slower by it than any other tile without parts of k;
* parts of k are at least four steps deep and none is empty."""
import ctypes
import math
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "pih_amd", "csrc")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    path = str(tmp_path_factory.mktemp("route") / "route.so")
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror", "-I", CSRC,
                    os.path.join(HERE, "dma_route_check.cpp"), "-o", path], check=True)
    lib = ctypes.CDLL(path)
    lib.route.restype = lib.rows_us.restype = ctypes.c_float
    return lib


def _route(lib, m, n, k):
    out = (ctypes.c_uint32 * 3)()
    us = lib.route(m, n, k, out)
    return (*out, us)


ROWS = (1, 33, 64, 65, 128, 129, 255, 256, 257, 300, 512, 515, 1021, 2048, 4099)
COLUMNS = (64, 200, 256, 1024, 4096, 24576)


@pytest.mark.parametrize("k", [64, 128, 192, 256, 320, 512, 1024, 4160, 24576])
def test_estimates_and_parts(lib, k):
    for m in ROWS:
        for n in COLUMNS:
            whole, rows, splits, us = _route(lib, m, n, k)
            assert math.isfinite(us), (m, n, k)
            assert whole % 256 == 0 and whole < m and rows in (64, 128, 256)
            steps = k // 64
            part = -(-steps // splits)
            assert splits == 1 or (steps // splits >= 4 and -(-steps // part) == splits)
            for r in (64, 128, 256):
                # (or as long as the weights take at their rate on the CUs in use)
                tiles = -(-m // r) * -(-n // 256)
                weights = n * k * 2 / 5.1e6 / (min(tiles, 256) / 256)
                assert us <= max(lib.rows_us(m, n, k, 1, r), weights) * 1.0001, (m, n, k, r)


@pytest.mark.parametrize("k", [64, 128, 192])
def test_few_rows_of_few_steps_take_low_tiles(lib, k):
    """One step's time of a tile of 64 rows is half that of one of 256."""
    for m in (1, 33, 64):
        for n in COLUMNS:
            assert _route(lib, m, n, k)[:3] == (0, 64, 1)
