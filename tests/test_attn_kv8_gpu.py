"""Attention over the paged 8-bit cache against the formula in 64 bits.

The tolerance of an output element: its rounding to the output type, plus, on
sum_j p_j |v_j|, the rounding of each weight to fp16 (2^-11) and twice the
relative error that an error in the scores gives the weights.  A score is a sum
of head_dim products in fp32, times two factors: (head_dim + 8) 2^-24 of the
sum of the products' magnitudes; exp adds 2^-20."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kernels_b200 as kb
from kv_ref import DTYPES, ROUND, attention, f64, filled_cache, values

pytestmark = pytest.mark.gpu


def run_case(start, new, Hq, H, D, bt, fmt, dtype, window, with_sinks, seed=0, qscale=1.0):
    rng = np.random.default_rng(seed)
    lens = [s + n for s, n in zip(start, new)]
    cpu, table = filled_cache(lens, H, D, bt, fmt, rng)
    dev = kb.KVCache(*(cpu[x].cuda() for x in ("k", "v", "k_scale", "v_scale")))
    T = sum(new)
    q = torch.from_numpy(rng.normal(0, qscale, (T, Hq, D)).astype(np.float32)).to(DTYPES[dtype])
    sinks = rng.normal(0, 2, Hq).astype(np.float32) if with_sinks else None
    i32 = dict(dtype=torch.int32, device="cuda")
    r = kb.kv_range(table.cuda(), torch.tensor(start, **i32),
                    torch.tensor([0] + list(np.cumsum(new)), **i32), max(new), max(lens))
    scale = D ** -0.5
    P = kb.attn_params(Hq, DTYPES[dtype], scale=scale, window=window)
    ws = kb.AttnWorkspace(dev, r, P)
    qd = q.cuda()
    out = torch.full_like(qd, float("nan"))
    lse = torch.full((T, Hq), float("nan"), device="cuda")
    sd = None if sinks is None else torch.from_numpy(sinks).cuda()
    kb.kv_device_errors(clear=True)
    kb.attn_kv8(dev, qd, out, r, P, ws, sinks=sd, lse=lse)
    assert not any(kb.kv_device_errors().values())
    at = 0
    for b, (s, n) in enumerate(zip(start, new)):
        if n:
            K, V = (values(cpu, x, table, b, s + n, bt) for x in ("k", "v"))
            o, l, a, mag = attention(f64(q[at:at + n]), K, V, s, np.float64(np.float32(scale)),
                                     window, None if sinks is None else sinks.astype(np.float64))
            d = (D + 8) * 2.0 ** -24 * mag + 2.0 ** -20
            tol = ROUND[dtype] * abs(o) * 1.01 + a * (2.0 ** -11 + 2 * d) + 1e-7
            got = f64(out[at:at + n])
            assert np.isfinite(got).all()
            worst = (abs(got - o) / tol).max()
            assert worst <= 1, f"sequence {b}: {worst} of the tolerance"
            gl = lse[at:at + n].cpu().double().numpy()
            assert (abs(gl - l) <= d + 2.0 ** -20 * (1 + abs(l))).all()
        at += n
    # the same call gives the same bits
    again, lse2 = torch.empty_like(out), torch.empty_like(lse)
    kb.attn_kv8(dev, qd, again, r, P, ws, sinks=sd, lse=lse2)
    assert torch.equal(again, out) and torch.equal(lse2, lse)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads", [(64, 8, 64), (32, 8, 128), (1, 1, 16), (10, 2, 96), (16, 1, 80),
                                   (3, 3, 256), (34, 2, 64)])
def test_single_tokens(lib, heads, dtype, fmt):
    Hq, H, D = heads
    run_case([0, 1, 15, 16, 63, 64, 200, 701], [1] * 8, Hq, H, D, 16, fmt, dtype, 0, True)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bt", [16, 32, 64, 128])
@pytest.mark.parametrize("window", [0, 1, 37, 128, 100000])
def test_windows_and_blocks(lib, bt, fmt, window):
    run_case([0, 130, 389, 1023], [3, 1, 2, 5], 8, 2, 64, bt, fmt, "f16", window, bt == 32)


@pytest.mark.parametrize("shape", [
    # start, new, q heads, heads, dim
    ([0], [1], 8, 8, 64), ([0], [130], 16, 2, 64), ([0, 700], [129, 64], 8, 1, 128),
    ([300, 0, 5], [17, 0, 33], 20, 4, 64), ([64], [200], 3, 1, 96), ([31, 9], [16, 257], 5, 1, 256),
    ([1000], [65], 128, 8, 64), ([2], [9], 32, 1, 48)])
@pytest.mark.parametrize("window,sinks", [(0, False), (50, True)])
def test_several_tokens(lib, shape, window, sinks):
    start, new, Hq, H, D = shape
    run_case(start, new, Hq, H, D, 32, "int8", "bf16", window, sinks, seed=5)
    run_case(start, new, Hq, H, D, 16, "e4m3", "f16", window, sinks, seed=6)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_long_context(lib, fmt):
    run_case([40001, 7], [1, 1], 16, 2, 64, 64, fmt, "f16", 0, False, seed=1, qscale=2.0)
    run_case([30000], [2], 16, 1, 128, 128, fmt, "bf16", 4000, True, seed=2, qscale=2.0)


def test_many_sequences(lib):
    n = 150
    run_case([(i * 53) % 300 for i in range(n)], [1 + (i % 7 == 0) for i in range(n)], 8, 2, 64, 16,
             "int8", "f16", 0, True, seed=3)
    run_case([(i * 53) % 300 for i in range(n)], [1] * n, 4, 1, 64, 16, "e4m3", "bf16", 64, False,
             seed=4)


def test_sharp_scores(lib):
    """One key takes all the weight; scores in the hundreds."""
    run_case([500], [1], 8, 1, 64, 16, "int8", "f16", 0, False, seed=7, qscale=300.0)
    run_case([500], [40], 8, 1, 64, 16, "int8", "bf16", 0, True, seed=7, qscale=300.0)


def cache_of(K, V, bt=16, fmt=torch.int8):
    T, H, D = K.shape
    nb = -(-T // bt)
    dev = kb.KVCache.empty(nb + 1, H, D, bt, dtype=fmt)
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.arange(nb, 0, -1, **i32)[None]
    kb.kv_write(dev, K, V, kb.kv_range(table, torch.zeros(1, **i32), torch.tensor([0, T], **i32), T, T))
    return dev, table


def one_range(table, start, n, longest=None):
    i32 = dict(dtype=torch.int32, device="cuda")
    return kb.kv_range(table, torch.tensor([start], **i32), torch.tensor([0, n], **i32), n,
                       longest or start + n)


def attend(dev, q, r, P, **kw):
    out = torch.empty_like(q)
    kb.attn_kv8(dev, q, out, r, P, kb.AttnWorkspace(dev, r, P), **kw)
    return out


def test_scales_far_apart(lib):
    """Blocks whose scales differ by many orders, blocks of zeros among them."""
    g = torch.Generator(device="cuda").manual_seed(0)
    T, H, D = 160, 1, 64
    K = torch.randn(T, H, D, device="cuda", generator=g)
    V = torch.randn(T, H, D, device="cuda", generator=g)
    for j, f in enumerate([1.0, 0.0, 1e-8, 1e6, 1e-3, 0.0, 1.0, 1e-12, 30.0, 1e-15]):
        V[16 * j:16 * j + 16] *= f
    V[48:64, :, ::2] = 0
    dev, table = cache_of(K, V)
    q = torch.randn(3, 8, D, device="cuda", generator=g).to(torch.bfloat16)
    P = kb.attn_params(8, torch.bfloat16, scale=0.125)
    lse = torch.empty(3, 8, device="cuda")
    out = attend(dev, q, one_range(table, T - 3, 3), P, lse=lse)
    k, v = (torch.empty(T, H, D, device="cuda") for _ in "kv")
    kb.kv_read(dev, k, v, one_range(table, 0, T))
    o, l, a, mag = attention(f64(q), f64(k), f64(v), T - 3, 0.125, 0, None)
    d = (D + 8) * 2.0 ** -24 * mag + 2.0 ** -20
    assert (abs(f64(out) - o) <= ROUND["bf16"] * abs(o) * 1.01 + a * (2.0 ** -11 + 2 * d)).all()
    assert (abs(lse.cpu().double().numpy() - l) <= d + 2.0 ** -20 * (1 + abs(l))).all()


def test_one_key_returns_its_value(lib):
    K = torch.randn(40, 2, 64, device="cuda")
    V = torch.randn(40, 2, 64, device="cuda")
    dev, table = cache_of(K, V)
    v = [torch.empty(40, 2, 64, device="cuda", dtype=torch.float16) for _ in "kv"]
    kb.kv_read(dev, *v, one_range(table, 0, 40))
    q = torch.randn(40, 4, 64, device="cuda").to(torch.float16)
    out = attend(dev, q, one_range(table, 0, 40), kb.attn_params(4, scale=1.0, window=1))
    want = v[1].float().repeat_interleave(2, dim=1)
    # the weight and its sum are the same number but for their rounding
    assert ((out.float() - want).abs() <= 2.0 ** -10 * want.abs() + 1e-7).all()


def test_sinks_only_and_minus_infinity(lib):
    K = torch.zeros(16, 1, 64, device="cuda")
    V = torch.ones(16, 1, 64, device="cuda")
    dev, table = cache_of(K, V)
    q = torch.ones(1, 2, 64, device="cuda", dtype=torch.float16)
    P = kb.attn_params(2, scale=1.0)
    sinks = torch.tensor([-float("inf"), 100.0], device="cuda")
    lse = torch.empty(1, 2, device="cuda")
    out = attend(dev, q, one_range(table, 15, 1), P, sinks=sinks, lse=lse)
    assert ((out[0, 0].float() - 1).abs() <= 2.0 ** -10).all()
    assert (out[0, 1] == 0).all()
    assert abs(float(lse[0, 0]) - np.log(16)) <= 1e-5 and abs(float(lse[0, 1]) - 100) <= 1e-4


def test_nan_and_infinite_queries_stay_in_their_rows(lib):
    g = torch.Generator(device="cuda").manual_seed(0)
    K, V = (torch.randn(100, 2, 64, device="cuda", generator=g) for _ in "kv")
    dev, table = cache_of(K, V)
    for dt in (torch.float16, torch.bfloat16):
        for n in (2, 60):
            q = torch.randn(n, 4, 64, device="cuda", generator=g).to(dt)
            P = kb.attn_params(4, scale=0.125)
            want = attend(dev, q, one_range(table, 100 - n, n), P)
            q[1, 1, 5], q[0, 2, 0] = float("nan"), float("inf")
            got = attend(dev, q, one_range(table, 100 - n, n), P)
            assert torch.isnan(got[1, 1]).all() and torch.isnan(got[0, 2]).all()
            keep = torch.ones(n, 4, dtype=torch.bool)
            keep[1, 1] = keep[0, 2] = False
            assert torch.equal(got[keep], want[keep])


def test_large_bf16_queries(lib):
    """bf16 reaches beyond fp16's range, up and down."""
    g = torch.Generator(device="cuda").manual_seed(1)
    K, V = (torch.randn(90, 1, 64, device="cuda", generator=g) for _ in "kv")
    dev, table = cache_of(K, V)
    q = torch.randn(2, 8, 64, device="cuda", generator=g).to(torch.bfloat16)
    for f in (2.0 ** 30, 2.0 ** -30):
        P1, P2 = kb.attn_params(8, scale=0.125), kb.attn_params(8, scale=0.125 / f)
        a = attend(dev, q, one_range(table, 88, 2), P1)
        b = attend(dev, (q.float() * f).to(torch.bfloat16), one_range(table, 88, 2), P2)
        assert torch.equal(a, b)


def test_strided_queries_and_outputs(lib):
    g = torch.Generator(device="cuda").manual_seed(2)
    K, V = (torch.randn(70, 2, 64, device="cuda", generator=g) for _ in "kv")
    dev, table = cache_of(K, V)
    for n in (1, 3, 40):
        qkv = torch.randn(n, 8 * 64, device="cuda", generator=g).to(torch.float16)
        q = qkv[:, 2 * 64:6 * 64].view(n, 4, 64)
        r, P = one_range(table, 70 - n, n), kb.attn_params(4, scale=0.125)
        want = attend(dev, q.contiguous(), r, P)
        wide = torch.zeros(4, n, 128, device="cuda", dtype=torch.float16)
        kb.attn_kv8(dev, q, wide[:, :, 64:].transpose(0, 1), r, P, kb.AttnWorkspace(dev, r, P))
        assert torch.equal(wide[:, :, 64:].transpose(0, 1), want)
        assert (wide[:, :, :64] == 0).all()


def test_shared_blocks(lib):
    """Two sequences with a common prefix give what one of them gives alone."""
    g = torch.Generator(device="cuda").manual_seed(3)
    K, V = (torch.randn(64, 1, 64, device="cuda", generator=g) for _ in "kv")
    dev, table = cache_of(K, V)
    q = torch.randn(1, 8, 64, device="cuda", generator=g).to(torch.float16)
    P = kb.attn_params(8, scale=0.125)
    want = attend(dev, q, one_range(table, 63, 1), P)
    i32 = dict(dtype=torch.int32, device="cuda")
    r = kb.kv_range(table.repeat(3, 1), torch.tensor([63, 40, 63], **i32),
                    torch.arange(4, **i32), 1, 64)
    got = attend(dev, q.repeat(3, 1, 1), r, P)
    for b in (0, 2):
        assert (got[b] - want[0]).abs().max() <= 2.0 ** -9 * want.abs().max()


def test_bad_blocks_and_bounds_are_reported(lib):
    K = torch.randn(64, 1, 64, device="cuda")
    dev, table = cache_of(K, K)
    P = kb.attn_params(8, scale=0.125)
    q = torch.randn(4, 8, 64, device="cuda").to(torch.float16)
    for bad in (5, -1, 0x7FFFFFFF):
        t = table.clone()
        t[0, 1] = bad
        kb.kv_device_errors(clear=True)
        attend(dev, q[:1], one_range(t, 50, 1), P)
        assert kb.kv_device_errors(clear=True)["block"]
        q40 = q.repeat(10, 1, 1)
        attend(dev, q40, one_range(t, 20, 40), P)
        assert kb.kv_device_errors(clear=True)["block"]
    i32 = dict(dtype=torch.int32, device="cuda")
    for start, cu, most, longest in (([61], [0, 4], 4, 64), ([0], [0, 4], 3, 64),
                                     ([-2], [0, 4], 4, 64), ([0], [0, 5], 5, 64)):
        r = kb.kv_range(table, torch.tensor(start, **i32), torch.tensor(cu, **i32), most, longest)
        attend(dev, q, r, P)
        assert kb.kv_device_errors(clear=True) == {"block": False, "bounds": True, "wait": False}


def test_graph_other_stream_and_a_workspace_for_several_shapes(lib):
    g = torch.Generator(device="cuda").manual_seed(4)
    K, V = (torch.randn(3000, 2, 64, device="cuda", generator=g) for _ in "kv")
    dev, table = cache_of(K, V)
    P = kb.attn_params(16, scale=0.125)
    ranges = [one_range(table, 2999, 1, 3000), one_range(table, 200, 300, 3000),
              one_range(table, 2500, 4, 3000)]
    qs = [torch.randn(n, 16, 64, device="cuda", generator=g).to(torch.float16) for n in (1, 300, 4)]
    want = [attend(dev, q, r, P) for q, r in zip(qs, ranges)]
    ws = max((kb.AttnWorkspace(dev, r, P) for r in ranges), key=lambda w: w.nbytes)
    outs = [torch.zeros_like(q) for q in qs]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        for q, r, o in zip(qs, ranges, outs):
            kb.attn_kv8(dev, q, o, r, P, ws)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
            o.zero_()
    with torch.cuda.stream(s):
        kb.attn_kv8(dev, qs[1], outs[1], ranges[1], P, ws)
    s.synchronize()
    assert torch.equal(outs[1], want[1])


def test_offsets_beyond_32_bits(lib):
    """A cache of more than 4 GiB a side, its last blocks in use."""
    H, D, bt = 8, 128, 128
    n_blocks = (1 << 32) // (H * D * bt) + 64
    dev = kb.KVCache.empty(n_blocks, H, D, bt)
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.tensor([[n_blocks - 1, n_blocks - 3]], **i32)
    g = torch.Generator(device="cuda").manual_seed(5)
    T = 200
    K, V = (torch.randn(T, H, D, device="cuda", generator=g) for _ in "kv")
    kb.kv_write(dev, K, V, one_range(table, 0, T))
    small = kb.KVCache.empty(2, H, D, bt)
    t2 = torch.tensor([[1, 0]], **i32)
    kb.kv_write(small, K, V, one_range(t2, 0, T))
    assert torch.equal(dev.k[n_blocks - 1], small.k[1]) and torch.equal(dev.v[n_blocks - 3], small.v[0])
    for n in (1, 50):
        q = torch.randn(n, 32, D, device="cuda", generator=g).to(torch.float16)
        P = kb.attn_params(32, scale=D ** -0.5)
        a = attend(dev, q, one_range(table, T - n, n), P)
        b = attend(small, q, one_range(t2, T - n, n), P)
        assert torch.equal(a, b)
    del dev
    torch.cuda.empty_cache()
