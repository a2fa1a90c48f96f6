"""Rotary positions against the formula in 64 bits.

Sine and cosine are off by 2^-20 (16-bit types: the device's approximate ones, 2^-21, of an
angle to 2^-24 of a turn, 2^-21.3) or 2^-22 (fp32: an angle to 2^-25 of half a turn, 2^-23.3, and
2^-23 of the functions), each acting on one of the pair's elements; the two products and their
sum are rounded three times (2^-24 each).  Then the result is rounded to its type."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

import kernels_b200 as kb
from draft_ref import frequencies, rotate
from kv_ref import DTYPES, ROUND, f64

pytestmark = pytest.mark.gpu
SINE = {"f16": 2.0 ** -20, "bf16": 2.0 ** -20, "f32": 2.0 ** -22}
SCALED = {"plain": {}, "linear": dict(factor=3.0), "yarn": dict(factor=32.0, orig_len=4096.0),
          "bands": dict(factor=8.0, orig_len=8192.0, low=1.0, high=4.0)}


def check(got, x, pos, f, layout, dtype, amplitude=1.0, inverse=False):
    y, mag = rotate(f64(x), pos, f, layout, amplitude, inverse)
    tol = ROUND[dtype] * abs(y) * 1.001 + mag * (SINE[dtype] + 3 * 2.0 ** -24) + 2.0 ** -25 * (dtype == "f16")
    err = abs(f64(got) - y)
    assert (err <= tol).all(), float((err / np.maximum(tol, 1e-300)).max())


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", [(1, 1, 16, 16), (3, 5, 64, 64), (17, 72, 64, 32), (2, 9, 96, 96),
                                   (300, 40, 128, 48), (33, 3, 256, 256), (5000, 10, 80, 16)])
def test_against_the_formula(lib, shape, layout, dtype):
    T, H, D, n = shape
    rng = np.random.default_rng(T)
    wide = torch.from_numpy(rng.normal(0, 2, (T, H + 3, D)).astype(np.float32)).to(DTYPES[dtype]).cuda()
    x = wide[:, 1:H + 1]                       # a slice of a wider buffer
    pos = rng.integers(0, 200000, T).astype(np.int32)
    table = kb.RopeTable(n, base=150000.0, layout=layout)
    out = torch.full((T, H, D), float("nan"), dtype=DTYPES[dtype], device="cuda")
    p = torch.from_numpy(pos).cuda()
    kb.rope(x, out, p, table)
    check(out, x, pos, frequencies(n, 150000.0), layout, dtype)
    assert torch.equal(out[..., n:], x[..., n:])
    # in place, and nothing beside the slice
    before = wide.clone()
    kb.rope(x, x, p, table)
    assert torch.equal(x, out)
    assert torch.equal(wide[:, 0], before[:, 0]) and torch.equal(wide[:, H + 1:], before[:, H + 1:])


@pytest.mark.parametrize("scaling", list(SCALED))
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_scalings_and_far_positions(lib, scaling, dtype):
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.normal(0, 1, (12, 4, 64)).astype(np.float32)).to(DTYPES[dtype]).cuda()
    pos = np.array([0, 1, -1, 7, 4095, 131071, 131072, 1 << 20, 16777217, 2 ** 31 - 1, -2 ** 31, -77],
                   np.int32)
    table = kb.RopeTable(64, base=500000.0, scaling=scaling, amplitude=1.25, **SCALED[scaling])
    out = torch.empty_like(x)
    kb.rope(x, out, torch.from_numpy(pos).cuda(), table)
    # (2^31 positions of a frequency that is held to 2^-53 of a turn and of its own 64-bit error:
    # 2^-20 of a turn at most)
    y, mag = rotate(f64(x), pos, frequencies(64, 500000.0, scaling, **SCALED[scaling]), "half", 1.25)
    far = np.abs(pos.astype(np.float64))[:, None, None] * 2.0 ** -50
    tol = ROUND[dtype] * abs(y) * 1.001 + mag * (SINE[dtype] + 2.0 ** -22 + far) + 2.0 ** -25
    assert (abs(f64(out) - y) <= tol).all()


def test_own_frequencies_and_more_than_a_turn(lib):
    rng = np.random.default_rng(2)
    f = np.concatenate([rng.uniform(-20, 20, 6), [0.0, 2 * np.pi]])
    x = torch.from_numpy(rng.normal(0, 1, (9, 2, 32)).astype(np.float32)).cuda()
    pos = np.arange(-4, 5).astype(np.int32)
    table = kb.RopeTable(16, layout="interleaved", freqs=torch.from_numpy(f).cuda())
    out = torch.empty_like(x)
    kb.rope(x, out, torch.from_numpy(pos).cuda(), table)
    check(out, x, pos, f, "interleaved", "f32")


def test_turning_back_is_the_gradient(lib):
    """<rope(x), g> has the gradient rope(g, inverse) in x; turned there and back a
    vector is itself times amplitude^2."""
    g = torch.Generator(device="cuda").manual_seed(0)
    x, d = (torch.randn(40, 6, 64, device="cuda", generator=g) for _ in range(2))
    pos = torch.arange(40, device="cuda", dtype=torch.int32) * 321
    for layout in ("half", "interleaved"):
        table = kb.RopeTable(48, layout=layout, amplitude=1.5)
        y, dx, back = (torch.empty_like(x) for _ in range(3))
        kb.rope(x, y, pos, table)
        kb.rope(d, dx, pos, table, inverse=True)
        check(dx, d, pos.cpu().numpy(), frequencies(48), layout, "f32", 1.5, True)
        # differences: the map is linear, so any step gives the derivative
        a, b = (y.double() * d.double()).sum(), (x.double() * dx.double()).sum()
        mag = (x.abs() @ d.abs().transpose(1, 2)).double().sum()
        assert abs(a - b) <= mag * 2.0 ** -20
        kb.rope(y, back, pos, table, inverse=True)
        # two turns' errors of 1.5 (2^-22 + 3 2^-24) on a pair's magnitudes, the second after a factor 1.5
        assert (back[..., :48] - 2.25 * x[..., :48]).abs().max() <= 2 * 2.25 * 2 * x.abs().max() * 2.0 ** -21
        assert torch.equal(back[..., 48:], x[..., 48:])


def test_strides_nothing_and_graphs(lib):
    table = kb.RopeTable(32)
    x = torch.randn(8, 7, 64, device="cuda").half().transpose(0, 1)      # heads outside tokens
    out = torch.empty(8, 7, 64, device="cuda", dtype=torch.half).transpose(0, 1)
    pos = torch.arange(7, device="cuda", dtype=torch.int32) + 1000
    kb.rope(x, out, pos, table)
    check(out, x, pos.cpu().numpy(), frequencies(32), "half", "f16")
    kb.rope(x[:0], out[:0], pos[:0], table)
    kb.rope(x[:, :0], out[:, :0], pos, table)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = torch.empty_like(out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        kb.rope(x, got, pos, table)
    pos += 5
    kb.rope(x, out, pos, table)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, out)


def test_broadcast_input(lib):
    """One row for every token, one head for every head."""
    x = torch.randn(1, 1, 64, device="cuda").expand(9, 5, 64)
    out = torch.empty(9, 5, 64, device="cuda")
    pos = torch.arange(9, device="cuda", dtype=torch.int32)
    kb.rope(x, out, pos, kb.RopeTable(64))
    check(out, x, np.arange(9), frequencies(64), "half", "f32")


def test_infinities_stay_in_their_pair(lib):
    x = torch.randn(2, 1, 64, device="cuda").half()
    x[0, 0, 3], x[1, 0, 40] = float("inf"), float("nan")
    out = torch.empty_like(x)
    kb.rope(x, out, torch.tensor([5, 6], device="cuda", dtype=torch.int32), kb.RopeTable(64))
    bad = ~torch.isfinite(out[:, 0])
    assert bad[0].nonzero().flatten().tolist() == [3, 35] and bad[1].nonzero().flatten().tolist() == [8, 40]
