"""CPU: the attention kernels' split of the work, compiled for the host, against
sums taken one by one (signed overflow wraps, as it does in the kernels)."""
from __future__ import annotations

import ctypes as C
import random
import subprocess

import pytest

from conftest import ROOT

SOURCE = r'''
#include "attn_split.cuh"
using namespace graft::dev;
extern "C" long long keys(int start, int n, int tt, int tiles, int rt, int window, int pad) {
    return tile_keys(start, n, tt, tiles, rt, window, pad);
}
'''


@pytest.fixture(scope="module")
def split(tmp_path_factory):
    d = tmp_path_factory.mktemp("split")
    (d / "s.cpp").write_text(SOURCE)
    so = d / "s.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fwrapv", "-shared", "-fPIC",
                    "-I", str(ROOT / "kernels_b200" / "csrc"), str(d / "s.cpp"), "-o", str(so)],
                   check=True)
    lib = C.CDLL(str(so))
    lib.keys.restype = C.c_longlong
    return lib


INT_MAX = 2 ** 31 - 1


@pytest.mark.parametrize("window", [0, 1, 2, 31, 32, 33, 100, 5000, 1 << 20, 1 << 30, INT_MAX - 255,
                                    INT_MAX - 40, INT_MAX - 1, INT_MAX])
def test_keys_of_row_tiles(split, window):
    rng = random.Random(window)
    cases = [(0, 200, 32), (0, 1, 1), (1 << 30, 0, 256), ((1 << 30) - 300, 300, 51), (0, 33, 256)]
    cases += [(rng.choice([0, rng.randrange(10000), rng.randrange(1 << 29)]), rng.randrange(1, 2000),
               rng.choice([1, 2, 32, 51, 128, 256])) for _ in range(60)]
    for start, n, tt in cases:
        tiles, pad, total = -(-n // tt), rng.choice([0, 192, 384]), 0
        for rt in range(tiles + 1):
            assert split.keys(start, n, tt, tiles, rt, window, pad) == total, (start, n, tt, rt)
            if rt < tiles:
                first = start + rt * tt
                k0 = first - window + 1 if window and first >= window else 0
                total += start + min(n, (rt + 1) * tt) - k0 + pad
