"""The cache write that turns its keys: every stored key is within half a step of the
turned key in 64 bits (the turn itself as in test_rope_gpu.py), values are stored exactly as
kv_write does, queries are turned exactly as rope does."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kernels_b200 as kb
from draft_ref import frequencies, rotate
from kv_ref import DTYPES, QMAX, filled_cache, f64
from test_kv_cache_gpu import half_step, rng_of, to_dev
from test_rope_gpu import SINE

pytestmark = pytest.mark.gpu

CASES = [
    # starts, new tokens, heads, dim, block, turned dims, query heads
    ([0], [1], 1, 16, 16, 16, 1),
    ([5, 16, 31], [1, 1, 1], 8, 128, 16, 64, 32),
    ([0, 0, 0], [64, 65, 63], 2, 64, 64, 64, 16),
    ([5, 0, 77], [40, 0, 131], 3, 96, 32, 48, 3),
    ([127], [2], 1, 256, 128, 256, 4),
    ([3, 128], [300, 128], 2, 256, 128, 32, 2),
    (list(range(0, 140, 2)), [1 + i % 3 for i in range(70)], 2, 80, 16, 80, 20),
    (list(range(160)), [1 + i % 8 for i in range(160)], 8, 64, 64, 64, 0),
    ([60, 9], [500, 1300], 4, 64, 64, 64, 32),
]


def stored(dev, x, table, b, lo, hi, bt):
    """Codes and scales of positions lo .. hi - 1: [n, heads, dim] and [n, heads, 1]."""
    codes, scale = getattr(dev, x).cpu(), getattr(dev, x + "_scale").cpu()
    blk = table[b].long()[torch.arange(lo, hi) // bt]
    c = codes.view(torch.uint8)[blk, :, torch.arange(lo, hi) % bt].view(codes.dtype)
    return c.float().double().numpy(), scale[blk].double().numpy()[:, :, None]


def check_keys(dev, cpu, table, b, lo, turned, mag, dtype, fmt, bt):
    """The stored keys of positions lo.. against fp64 ones."""
    hi = lo + len(turned)
    code, scale = stored(dev, "k", table, b, lo, hi, bt)
    err = (SINE[dtype] + 3 * 2.0 ** -24) * mag + 2.0 ** -22 * abs(turned)
    step = scale * np.maximum(half_step(code, fmt), half_step(turned / scale, fmt))
    assert (abs(code * scale - turned) <= step + err).all()
    # each block's scale: the largest magnitude of its new keys, or what it was
    for j in range(lo // bt, -(-hi // bt)):
        at = slice(max(lo, j * bt) - lo, min(hi, (j + 1) * bt) - lo)
        blk = int(table[b, j])
        most = abs(turned[at]).max(axis=(0, 2)) / QMAX[fmt]
        slack = err[at].max(axis=(0, 2)) / QMAX[fmt] + 2.0 ** -23 * most
        got = dev.k_scale[blk].cpu().double().numpy()
        want = np.maximum(most, 2.0 ** -64)
        if j * bt < lo:
            want = np.maximum(want, cpu["k_scale"][blk].double().numpy())
        assert (abs(got - want) <= slack).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_write(lib, case, layout, dtype, fmt):
    start, new, H, D, bt, n, Hq = CASES[case]
    rng = np.random.default_rng(case)
    cpu, table = filled_cache([s + m for s, m in zip(start, new)], H, D, bt, fmt, rng)
    dev, plain = to_dev(cpu), to_dev(cpu)
    T = sum(new)
    qkv = torch.from_numpy(rng.normal(0, 1, (T, Hq + 2 * H, D)).astype(np.float32)).to(DTYPES[dtype]).cuda()
    qkv[:, Hq] *= 20          # a head whose scale grows
    q, K, V = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
    r = rng_of(table, start, new, extra=case % 3)
    rope = kb.RopeTable(n, base=150000.0, layout=layout, amplitude=1.1)
    pos = np.concatenate([np.arange(s, s + m) for s, m in zip(start, new)]).astype(np.int32)
    given = case % 2 == 1     # positions of their own
    if given:
        pos = rng.integers(0, 100000, T).astype(np.int32)
    out = torch.full((T, Hq, D), float("nan"), dtype=DTYPES[dtype], device="cuda")
    p = torch.from_numpy(pos).cuda()
    kb.kv_device_errors(clear=True)
    kb.kv_write_rope(dev, K, V, r, rope, positions=p if given else None,
                     **(dict(q=q, q_out=out) if Hq else {}))
    assert not any(kb.kv_device_errors().values())
    kb.kv_write(plain, K, V, r)
    assert torch.equal(dev.v.view(torch.uint8), plain.v.view(torch.uint8))
    assert torch.equal(dev.v_scale.view(torch.int32), plain.v_scale.view(torch.int32))
    if Hq:
        want = torch.empty_like(out)
        kb.rope(q, want, p, rope)
        assert torch.equal(out, want)
    turned, mag = rotate(f64(K), pos, frequencies(n, 150000.0), layout, 1.1)
    at = 0
    for b, (s, m) in enumerate(zip(start, new)):
        if m:
            check_keys(dev, cpu, table, b, s, turned[at:at + m], mag[at:at + m], dtype, fmt, bt)
            # earlier tokens of the first block: rounded again to the grown scale
            code, scale = stored(dev, "k", table, b, s - s % bt, s, bt)
            if s % bt:
                blk = int(table[b, s // bt])
                old = (cpu["k"][blk].float().double().numpy()[:, :s % bt].transpose(1, 0, 2) *
                       cpu["k_scale"][blk].double().numpy()[None, :, None])
                step = scale * np.maximum(half_step(code, fmt), half_step(old / scale, fmt))
                assert (abs(code * scale - old) <= step * (1 + 1e-6) + 1e-30).all()
        at += m
    # blocks of no sequence stay as they are
    used = {int(table[b, j]) for b, (s, m) in enumerate(zip(start, new)) if m
            for j in range(s // bt, -(-(s + m) // bt))}
    rest = [i for i in range(len(cpu["k"])) if i not in used]
    assert torch.equal(dev.k.cpu().view(torch.uint8)[rest], cpu["k"].view(torch.uint8)[rest])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_rows_of_a_tree(lib, dtype, fmt):
    """Parts of each sequence's rows, in another order, one row twice, none at all."""
    start, new, bt, H, D = [5, 0, 31, 64, 7], [24, 33, 1, 40, 9], 16, 2, 64
    count, rng = [7, 33, 1, 20, 0], np.random.default_rng(0)
    cpu, table = filled_cache([s + m for s, m in zip(start, new)], H, D, bt, fmt, rng)
    T, cu = sum(new), np.cumsum([0] + new)
    K, V = (torch.from_numpy(rng.normal(0, 1, (T, H, D)).astype(np.float32)).to(DTYPES[dtype]).cuda()
            for _ in "kv")
    rows = np.full(T, -7, np.int32)
    for b, m in enumerate(count):
        rows[cu[b]:cu[b] + m] = cu[b] + np.sort(rng.permutation(new[b])[:m])
    rows[cu[3] + 4] = rows[cu[3] + 3]
    pos = rng.integers(0, 5000, T).astype(np.int32)
    rope = kb.RopeTable(64)
    r = rng_of(table, start, new)
    i32 = dict(dtype=torch.int32, device="cuda")
    for given in (True, False):
        dev, plain = to_dev(cpu), to_dev(cpu)
        kb.kv_device_errors(clear=True)
        kb.kv_write_rope(dev, K, V, r, rope, positions=torch.from_numpy(pos).cuda() if given else None,
                         rows=torch.from_numpy(rows).cuda(), count=torch.tensor(count, **i32))
        assert not any(kb.kv_device_errors().values())
        some = torch.from_numpy(np.concatenate([rows[cu[b]:cu[b] + m] for b, m in enumerate(count)])).cuda().long()
        kb.kv_write(plain, K[some], V[some], rng_of(table, start, count))
        assert torch.equal(dev.v.view(torch.uint8), plain.v.view(torch.uint8))
        for b, m in enumerate(count):
            if m:
                at = rows[cu[b]:cu[b] + m]
                p = pos[at] if given else np.arange(start[b], start[b] + m)
                turned, mag = rotate(f64(K)[at], p, frequencies(64), "half")
                check_keys(dev, cpu, table, b, start[b], turned, mag, dtype, fmt, bt)
        blk = int(table[4, 0])     # a sequence that keeps nothing: untouched
        assert torch.equal(dev.k[blk].cpu().view(torch.uint8), cpu["k"][blk].view(torch.uint8))


def test_bad_rows_and_counts_are_reported(lib):
    cpu, table = filled_cache([40, 40], 1, 64, 16, "int8", np.random.default_rng(0))
    K = torch.randn(80, 1, 64, device="cuda").half()
    r, rope = rng_of(table, [0, 0], [40, 40]), kb.RopeTable(64)
    i32 = dict(dtype=torch.int32, device="cuda")
    rows = torch.arange(80, **i32)
    for bad, count in ((80, [3, 3]), (-1, [3, 3]), (2, [41, 3]), (2, [-1, 3])):
        dev = to_dev(cpu)
        rows[2] = bad
        kb.kv_device_errors(clear=True)
        kb.kv_write_rope(dev, K, K, r, rope, rows=rows, count=torch.tensor(count, **i32))
        assert kb.kv_device_errors(clear=True) == {"block": False, "bounds": True, "wait": False}
        blk = int(table[0, 0])
        if count[0] == 3:        # the row is written as zeros, the others as ever
            assert not dev.v[blk, 0, 2].any() and dev.v[blk, 0, 1].any()
        else:                    # the sequence is skipped
            assert torch.equal(dev.k[blk].cpu(), cpu["k"][blk])
        assert dev.v[int(table[1, 0]), 0, 2].any()


def test_infinities(lib):
    """A pair with an infinity or a NaN is stored as the formula has it: largest codes and 0."""
    cpu, table = filled_cache([2], 1, 64, 16, "int8", np.random.default_rng(0))
    dev = to_dev(cpu)
    K = torch.randn(2, 1, 64, device="cuda").half()
    K[0, 0, 3], K[1, 0, 40] = float("inf"), float("nan")
    kb.kv_write_rope(dev, K, K, rng_of(table, [0], [2]), kb.RopeTable(64),
                     positions=torch.tensor([1, 1], dtype=torch.int32, device="cuda"))
    k = dev.k[int(table[0, 0]), 0].cpu()
    # inf cos(1) and inf sin(1) are infinite (finite partners do not matter); NaN is 0
    assert k[0, 3] == 127 and k[0, 35] == 127 and k[1, 8] == 0 and k[1, 40] == 0
    assert torch.isfinite(dev.k_scale[int(table[0, 0])]).all()


def test_captured(lib):
    """Lengths, rows and counts follow the device's memory in a replay."""
    cpu, table = filled_cache([60], 2, 64, 16, "int8", np.random.default_rng(3))
    a, b = to_dev(cpu), to_dev(cpu)
    g = torch.Generator(device="cuda").manual_seed(0)
    K = torch.randn(30, 2, 64, device="cuda", generator=g).half()
    i32 = dict(dtype=torch.int32, device="cuda")
    start, cu = torch.tensor([10], **i32), torch.tensor([0, 30], **i32)
    count, rows, rope = torch.tensor([4], **i32), torch.arange(30, **i32), kb.RopeTable(64)
    r = kb.kv_range(table.cuda(), start, cu, 30, 60)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        kb.kv_write_rope(a, K, K, r, rope, rows=rows, count=count)
    start += 7
    count += 9
    rows += 3
    graph.replay()
    kb.kv_write_rope(b, K, K, r, rope, rows=rows, count=count)
    torch.cuda.synchronize()
    for x in ("k", "v", "k_scale", "v_scale"):      # (unused scales are NaN: bits)
        assert torch.equal(getattr(a, x).view(torch.uint8), getattr(b, x).view(torch.uint8))
