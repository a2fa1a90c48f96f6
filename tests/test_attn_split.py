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
template <typename T>
static Split<T> split(T U, int G, int pad, int snap) {
    Split<T> s;
    s.set(U, G, pad, snap);
    return s;
}
extern "C" int bound(int U, int G, int c) { return split(U, G, 0, 1).bound(c); }
extern "C" int at_least(int U, int G, int x) { return split(U, G, 0, 1).at_least(x); }
extern "C" void cuts(int U, int G, int pad, int snap, int p0, int p1, int* out) {
    split(U, G, pad, snap).cuts(p0, p1, out[0], out[1]);
}
extern "C" int snapped(int U, int G, int pad, int snap, int x, int p0, int p1) {
    return split(U, G, pad, snap).snapped(x, p0, p1);
}
extern "C" long long at_least64(long long U, int G, long long x) { return split(U, G, 0, 1).at_least(x); }
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
    lib.keys.restype = lib.at_least64.restype = C.c_longlong
    lib.at_least64.argtypes = [C.c_longlong, C.c_int, C.c_longlong]
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


def bounds(U, G):
    """Where the G shares of U units begin, and the end."""
    return [c * (U // G) + min(c, U % G) for c in range(G + 1)]


@pytest.mark.parametrize("U", [1, 147, 1000, 12345678, 1 << 30, (1 << 31) - 300, (1 << 31) - 41])
@pytest.mark.parametrize("G", [1, 2, 148, 295, 512])
def test_shares_and_their_first_at_or_beyond(split, U, G):
    if G > U:
        return
    b = bounds(U, G)
    rng = random.Random(U + G)
    for c in sorted({0, 1, G // 2, G - 1, G} & set(range(G + 1))):
        assert split.bound(U, G, c) == b[c]
    xs = {1, U, max(1, U - 1), U // 2 + 1} | {rng.randrange(1, U + 1) for _ in range(200)}
    xs |= {min(U, max(1, x + d)) for x in rng.sample(b, min(len(b), 40)) for d in (-1, 0, 1)}
    for x in xs:
        want = next(c for c in range(G + 1) if b[c] >= x)
        assert split.at_least(U, G, x) == want, x
        assert split.at_least64(U, G, x) == want, x
        assert split.at_least64(U << 20, G, x << 20) == next(
            c for c, y in enumerate(bounds(U << 20, G)) if y >= x << 20)


@pytest.mark.parametrize("pad,snap", [(24, 16), (384, 256), (0, 1)])
def test_pieces_of_pairs(split, pad, snap):
    """Every unit of every pair belongs to one piece, and the pieces of a cut pair are
    those that its CTAs find: the one before the first cut has the first."""
    rng = random.Random(pad)
    for trial in range(120):
        sizes = [pad + rng.choice([1, 3, rng.randrange(1, 60), rng.randrange(1, 4000)])
                 for _ in range(rng.randrange(1, 40))]
        base = rng.choice([0, (1 << 31) - 1 - pad - snap - sum(sizes)])   # (a pair of all before)
        if base:
            sizes = [base] + sizes
        U = sum(sizes)
        G = max(1, min(rng.choice([3, 148, 296, 512]),
                       max(len(sizes), (U - len(sizes) * pad) // snap)))
        edges, at = [], 0
        for n in sizes:
            edges.append((at, at + n))
            at += n
        b = bounds(U, G)
        start = []
        for x in b[:-1]:
            p0, p1 = next(e for e in edges if e[0] <= x < e[1])
            start.append(split.snapped(U, G, pad, snap, x, p0, p1))
        start.append(U)
        assert start[0] == 0 and start == sorted(start)
        for p0, p1 in edges:
            inside = [c for c in range(G) if p0 < start[c] < p1]
            out = (C.c_int * 2)()
            split.cuts(U, G, pad, snap, p0, p1, out)
            assert list(range(out[0], out[1] + 1)) == inside
            cuts = [start[c] for c in inside]
            assert len(set(cuts)) == len(cuts)
            if inside:
                assert cuts[0] - p0 >= pad + snap and p1 - cuts[-1] >= snap
                first = inside[0] - 1
                assert start[first] <= p0 and start[inside[0]] > p0
