"""Attention over the 8-bit cache where it can go wrong at the edges: windows without a
limit and blocks they have left behind, scores that rise from unit to unit, huge and far
apart ones, scales that are zero, negative or no numbers."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kernels_b200 as kb
from kv_ref import ROUND, attention, f64
from test_attn_kv8_gpu import attend, cache_of, one_range, run_case

pytestmark = pytest.mark.gpu

INT_MAX = 2 ** 31 - 1


@pytest.mark.parametrize("window", [INT_MAX, INT_MAX - 40, 1 << 30, 701, 700])
def test_windows_beyond_every_sequence(lib, window):
    """The largest int as "no limit": the same bits as no window, for few and many rows."""
    g = torch.Generator(device="cuda").manual_seed(0)
    for H, D in ((2, 64), (1, 128), (1, 256)):
        K, V = (torch.randn(700, H, D, device="cuda", generator=g) for _ in "kv")
        dev, table = cache_of(K, V)
        for start, n in ((699, 1), (690, 10), (0, 200), (300, 400)):
            q = torch.randn(n, 8 * H, D, device="cuda", generator=g).to(torch.float16)
            want = attend(dev, q, one_range(table, start, n), kb.attn_params(8 * H, scale=D ** -0.5))
            got = attend(dev, q, one_range(table, start, n),
                         kb.attn_params(8 * H, scale=D ** -0.5, window=window))
            assert torch.equal(got, want), (H, D, start, n)
    assert not any(kb.kv_device_errors().values())


def test_windows_beyond_the_sequences_of_a_longer_bound(lib):
    """A window that is within max_len and beyond what the sequences hold."""
    run_case([0, 700, 5], [129, 64, 300], 8, 1, 64, 16, "int8", "f16", 1200, False)


def raw_cache(kc, vc, ks, vs, bt):
    """A cache of one sequence from int8 code values kc, vc [T, H, D] and scales ks, vs
    [ceil(T / bt), H]; block 0 belongs to nobody."""
    T, H, D = kc.shape
    nb = -(-T // bt)
    dev = kb.KVCache.empty(nb + 1, H, D, bt)
    for codes, x in ((dev.k, kc), (dev.v, vc)):
        pad = torch.zeros(nb * bt, H, D, dtype=torch.int8)
        pad[:T] = x.to(torch.int8)
        codes[1:] = pad.view(nb, bt, H, D).transpose(1, 2).cuda()
    dev.k_scale[1:], dev.v_scale[1:] = ks.cuda(), vs.cuda()
    return dev, torch.arange(1, nb + 1, dtype=torch.int32, device="cuda")[None]


def check_against_formula(dev, table, q, T, scale, window=0):
    """Output and lse of the sequence's last tokens against the formula in 64 bits, with
    the tolerances of test_attn_kv8_gpu.py."""
    n, Hq, D = q.shape
    P = kb.attn_params(Hq, scale=scale, window=window)
    lse = torch.empty(n, Hq, device="cuda")
    out = attend(dev, q, one_range(table, T - n, n), P, lse=lse)
    k, v = (torch.empty(T, dev.heads, D, device="cuda") for _ in "kv")
    kb.kv_read(dev, k, v, one_range(table, 0, T))
    o, l, a, mag = attention(f64(q), f64(k), f64(v), T - n, np.float64(np.float32(scale)), window, None)
    d = (D + 8) * 2.0 ** -24 * mag + 2.0 ** -20
    tol = ROUND["f16" if q.dtype == torch.float16 else "bf16"] * abs(o) * 1.01 + a * (2.0 ** -11 + 2 * d) + 1e-7
    assert (abs(f64(out) - o) <= tol).all(), (abs(f64(out) - o) / tol).max()
    assert (abs(lse.cpu().double().numpy() - l) <= d + 2.0 ** -20 * (1 + abs(l))).all()
    assert not any(kb.kv_device_errors().values())


@pytest.mark.parametrize("D", [64, 48, 128, 256])
@pytest.mark.parametrize("step", [2.0, 5.0, 9.0, 11.0, 12.0, 13.0, 14.0, 17.0])
@pytest.mark.parametrize("keys", [32, 64, 128])
def test_scores_that_rise(lib, keys, step, D):
    """Scores that rise by `step` (log2) every `keys` keys, so that references follow in
    every unit, go up before one and follow within it, and outputs are rescaled twice in
    a row.  Rows of a tile differ in how steep theirs are, down to falling ones."""
    g = torch.Generator().manual_seed(int(step) + keys + D)
    T, Hq, n = 900, 8, 60
    runs = -(-T // keys)
    kc = torch.randint(-2, 3, (T, 1, D), generator=g).float()
    kc[:, 0, 0] = (torch.arange(T) // keys).float() * 4       # up to 112
    vc = torch.randint(-127, 128, (T, 1, D), generator=g).float()
    nb = -(-T // 16)
    ks = torch.full((nb, 1), 0.25)
    vs = 2.0 ** torch.randint(-2, 3, (nb, 1), generator=g).float()
    dev, table = raw_cache(kc, vc, ks, vs, 16)
    q = 0.05 * torch.randn(n, Hq, D, generator=g)
    steep = torch.tensor([1.0, 1.0, 0.9, 0.5, 0.1, 0.0, -0.5, -1.0])
    q[:, :, 0] = steep * (1 + 0.01 * torch.arange(n))[:, None]
    check_against_formula(dev, table, q.half().cuda(), T, step / 1.4426950408889634)
    assert runs * 4 <= 127


@pytest.mark.parametrize("n", [3, 60])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_scales_far_apart_many_rows_too(lib, n, D):
    """Blocks whose scales differ by many orders, blocks of zeros among them."""
    g = torch.Generator(device="cuda").manual_seed(0)
    T, H = 320, 1
    K = torch.randn(T, H, D, device="cuda", generator=g)
    V = torch.randn(T, H, D, device="cuda", generator=g)
    factors = [1.0, 0.0, 1e-8, 1e6, 1e-3, 0.0, 1.0, 1e-12, 30.0, 1e-15]
    for j in range(T // 16):
        V[16 * j:16 * j + 16] *= factors[j % 10]
    V[48:64, :, ::2] = 0
    dev, table = cache_of(K, V)
    q = torch.randn(n, 8, D, device="cuda", generator=g).to(torch.bfloat16)
    check_against_formula(dev, table, q, T, D ** -0.5)


def check_huge(n, D, exponent):
    """Scores of about 2^exponent (log2 units) whose neighbours are one step of fp32 apart
    from 2^25 on: S, S + 1 and S + 2 in three runs of 256 keys, S about 1.66e7 < 2^24 (sums
    of products are exact in fp32) and of every parity, times 2^(exponent - 24)."""
    g = torch.Generator().manual_seed(0)
    T = 768
    kc = torch.zeros(T, 1, D)
    kc[:, 0, :2] = 127
    kc[:, 0, 2] = torch.arange(T) // 256
    kc[:, 0, 3] = 1
    vc = torch.randint(-127, 128, (T, 1, D), generator=g).float()
    dev, table = raw_cache(kc, vc, torch.ones(T // 16, 1), torch.ones(T // 16, 1), 16)
    q = torch.zeros(n, 8, D)
    q[:, :, :2] = 65504
    q[:, :, 2] = 1
    q[:, :, 3] = torch.arange(8)
    q = q.half().cuda()
    P = kb.attn_params(8, scale=2.0 ** (exponent - 24) / 1.4426950408889634)
    lse = torch.empty(n, 8, device="cuda")
    out = attend(dev, q, one_range(table, T - n, n), P, lse=lse)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    # the weights are what rounded scores make of them, but weights: an average of values
    # (each weight is off by 2^-11, the output by 2^-11 more)
    assert (out.float().cpu() <= vc.amax(0) * (1 + 2.0 ** -10)).all()
    assert (out.float().cpu() >= vc.amin(0) * (1 + 2.0 ** -10)).all()
    # lse is the largest score, off by a few roundings, and at most log T above
    top = (f64(q) @ kc[:, 0].double().numpy().T * np.float64(np.float32(P.scale))).max(-1)
    assert (abs(lse.cpu().double().numpy() - top) <= 2.0 ** -20 * abs(top) + np.log(T)).all()
    assert not any(kb.kv_device_errors().values())


@pytest.mark.parametrize("D", [64, 48, 128, 256])
@pytest.mark.parametrize("exponent", [18, 20, 22, 24, 25, 26, 27, 28, 29, 30, 34, 40])
def test_huge_scores_many_rows(lib, exponent, D):
    check_huge(60, D, exponent)


@pytest.mark.parametrize("n,D", [(1, 64), (2, 64), (4, 64), (1, 48), (1, 128), (2, 128), (1, 256)])
@pytest.mark.parametrize("exponent", [18, 20, 22, 24, 25, 26, 27, 28, 29, 30, 34, 40])
def test_huge_scores_few_rows(lib, exponent, n, D):
    check_huge(n, D, exponent)


@pytest.mark.parametrize("scale", [-1.0, float("inf"), float("nan")])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_sequence_of_bad_scales_keeps_to_itself(lib, scale, D):
    """Key scales that no cache should hold: the call ends, other sequences are right."""
    g = torch.Generator(device="cuda").manual_seed(1)
    T, n, nb = 300, 60, 19
    dev = kb.KVCache.empty(2 * nb, 1, D, 16)
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.arange(2 * nb, **i32).view(2, nb)
    K, V = (torch.randn(2 * T, 1, D, device="cuda", generator=g) for _ in "kv")
    kb.kv_write(dev, K, V, kb.kv_range(table, torch.zeros(2, **i32), torch.tensor([0, T, 2 * T], **i32), T, T))
    dev.k_scale[3:nb:2] = scale
    q = (40 * torch.randn(2 * n, 8, D, device="cuda", generator=g)).to(torch.float16)
    P = kb.attn_params(8, scale=D ** -0.5)
    want = attend(dev, q[n:], one_range(table[1:], T - n, n), P)
    r = kb.kv_range(table, torch.tensor([T - n] * 2, **i32), torch.tensor([0, n, 2 * n], **i32), n, T)
    got = attend(dev, q, r, P)[n:]
    assert (got.float() - want.float()).abs().max() <= 2.0 ** -9 * want.abs().max()
    assert not any(kb.kv_device_errors().values())


@pytest.mark.parametrize("left", ["minus one", "another's block"])
@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("bt", [16, 32, 64, 128])
@pytest.mark.parametrize("H,D", [(2, 64), (1, 128), (1, 256), (1, 48)])
def test_blocks_before_the_window_are_not_needed(lib, H, D, bt, fmt, left):
    """A host that frees the blocks which a window has left behind puts anything into
    their table entries: the same bits come out, and nothing is reported."""
    g = torch.Generator(device="cuda").manual_seed(0)
    T, G = 700, 4
    nb = -(-T // bt)
    dev = kb.KVCache.empty(nb + 1, H, D, bt, dtype=fmt)
    for c, s in ((dev.k, dev.k_scale), (dev.v, dev.v_scale)):   # block 0: what nobody wrote
        c.view(torch.uint8)[0] = 0x7F
        s[0] = float("nan")
    table = torch.arange(nb, 0, -1, dtype=torch.int32, device="cuda")[None]
    K, V = (torch.randn(T, H, D, device="cuda", generator=g) for _ in "kv")
    kb.kv_write(dev, K, V, one_range(table, 0, T))
    for c in (dev.k, dev.v):          # nor the last block's rest
        if T % bt:
            c.view(torch.uint8)[1, :, T % bt:] = 0x7F
    kb.kv_device_errors(clear=True)
    for n in (1, 2, 70, 300):
        for window in (1, 5, 12, 16, 17, 40, 130):
            q = torch.randn(n, H * G, D, device="cuda", generator=g).to(torch.float16)
            P = kb.attn_params(H * G, scale=D ** -0.5, window=window)
            want = attend(dev, q, one_range(table, T - n, n), P)
            assert torch.isfinite(want).all()
            freed = table.clone()
            freed[0, :max(0, T - n - window + 1) // bt] = -1 if left == "minus one" else 0
            got = attend(dev, q, one_range(freed, T - n, n), P)
            assert not any(kb.kv_device_errors(clear=True).values()), (n, window)
            assert torch.equal(got, want), (n, window)


@pytest.mark.parametrize("n,D,below", [(n, D, b) for n, D in ((1, 64), (4, 64), (1, 128), (1, 256), (60, 128))
                                       for b in (10.3, 16.3, 23.3)] +
                         [(60, D, b) for D in (64, 48, 256) for b in (10.3, 16.3)])
@pytest.mark.parametrize("alike", [False, True])
def test_many_keys_far_below_the_largest(lib, alike, n, D, below):
    """One key of value zero takes the weight; the output is what thousands of others add,
    each `below` (log2) under it: down to 2^-17 of the largest (2^-24 where the reference is
    found first) their weights keep fp16's 11 bits, also where all are rounded alike."""
    g = torch.Generator().manual_seed(0)
    T, bt = 4000, 64
    kc = torch.zeros(T, 1, D)
    kc[7, 0, 0] = 100
    if not alike:
        kc[:, 0, 1:] = torch.randint(-1, 2, (T, D - 1), generator=g).float()
    vc = torch.randint(20, 128, (T, 1, D), generator=g).float()
    vc[7] = 0
    nb = -(-T // bt)
    dev, table = raw_cache(kc, vc, torch.ones(nb, 1), torch.full((nb, 1), 0.01), bt)
    q = torch.zeros(n, 8, D)
    q[:, :, 0] = 1 - 0.005 * torch.arange(8)
    q[:, :, 1:] = 0.01 * torch.randn(n, 8, D - 1, generator=g)
    check_against_formula(dev, table, q.half().cuda(), T, below / 100 / 1.4426950408889634)


@pytest.mark.parametrize("scale", [-0.125, 0.0])
@pytest.mark.parametrize("n,D", [(1, 64), (4, 64), (60, 64), (60, 128), (60, 256)])
def test_scales_that_are_not_positive(lib, n, D, scale):
    g = torch.Generator(device="cuda").manual_seed(2)
    T = 500
    K, V = (torch.randn(T, 1, D, device="cuda", generator=g) for _ in "kv")
    dev, table = cache_of(K, V)
    q = torch.randn(n, 8, D, device="cuda", generator=g).half()
    check_against_formula(dev, table, q, T, scale)
