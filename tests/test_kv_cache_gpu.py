"""Writing the paged 8-bit cache and reading it back, against the definition in
64 bits: scales are the rounded amax / qmax exactly, every stored value is
within half a step of its input, and reading is code * scale rounded once."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kernels_b200 as kb
from kv_ref import CODES, DTYPES, QMAX, filled_cache

pytestmark = pytest.mark.gpu


def to_dev(cache):
    return kb.KVCache(*(cache[x].cuda() for x in ("k", "v", "k_scale", "v_scale")))


def rng_of(table, start, new, extra=0):
    i32 = dict(dtype=torch.int32, device="cuda")
    return kb.kv_range(table.cuda(), torch.tensor(start, **i32),
                       torch.tensor([0] + list(np.cumsum(new)), **i32), max(new) + extra,
                       max(s + n for s, n in zip(start, new)) + extra)


def half_step(y, fmt):
    """Half the distance of neighbouring codes around y (in units of the scale)."""
    if fmt == "int8":
        return 0.5
    e = np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -20)))
    return 2.0 ** (np.maximum(e, -6.0) - 4.0)


# (starts, new tokens, heads, dim, block): ends inside a block, on it, one past
# it; single tokens; nothing; a head_dim that is no power of two; many sequences
CASES = [
    ([0], [1], 1, 16, 16),
    ([0, 0, 0], [64, 65, 63], 2, 64, 64),
    ([5, 16, 31], [1, 1, 1], 8, 128, 16),
    ([5, 0, 77], [40, 0, 131], 3, 96, 32),
    ([127], [2], 1, 256, 128),
    ([0, 128], [300, 128], 2, 256, 128),
    (list(range(0, 140, 2)), [1 + i % 3 for i in range(70)], 2, 80, 16),
    (list(range(160)), [1 + i % 8 for i in range(160)], 8, 64, 64),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_write_then_read(lib, case, dtype, fmt):
    start, new, H, D, bt = CASES[case]
    rng = np.random.default_rng(case)
    lens = [s + n for s, n in zip(start, new)]
    cpu, table = filled_cache(lens, H, D, bt, fmt, rng)
    dev = to_dev(cpu)
    T = sum(new)
    x = {c: torch.from_numpy(rng.normal(0, 1, (T, H, D)).astype(np.float32)).to(DTYPES[dtype])
         for c in ("k", "v")}
    x["v"][:, 0] *= 50        # a head whose scale grows, one whose scale stays
    r = rng_of(table, start, new)
    kb.kv_device_errors(clear=True)
    kb.kv_write(dev, x["k"].cuda(), x["v"].cuda(), r)
    out = [torch.full((T, H, D), float("nan"), dtype=DTYPES[dtype], device="cuda") for _ in "kv"]
    kb.kv_read(dev, *out, r)
    assert not any(kb.kv_device_errors().values())
    for c, got in zip(("k", "v"), out):
        codes, scale = getattr(dev, c).cpu(), getattr(dev, c + "_scale").cpu()
        stored, were = codes.float().double().numpy(), cpu[c].float().double().numpy()
        s_new, s_was = scale.double().numpy(), cpu[c + "_scale"].double().numpy()
        xs = x[c].float().double().numpy()
        touched = np.zeros(len(codes), bool)
        at = 0
        for b, (s, n) in enumerate(zip(start, new)):
            for j in range(s // bt, -(-(s + n) // bt) if n else s // bt):
                blk = int(table[b, j])
                touched[blk] = True
                lo, hi = max(s, j * bt), min(s + n, (j + 1) * bt)
                part = xs[at + lo - s:at + hi - s].transpose(1, 0, 2)     # [H, tokens, D]
                want = np.float32(np.maximum(np.abs(part).max((1, 2)) / QMAX[fmt], 2.0 ** -64))
                held = lo - j * bt
                if held:
                    want = np.maximum(want, np.float32(s_was[blk]))
                assert np.array_equal(np.float32(s_new[blk]), want)
                y = part / s_new[blk][:, None, None]
                err = np.abs(stored[blk][:, held:hi - j * bt] - y)
                assert (err <= half_step(y, fmt) * (1 + 2.0 ** -20) + 2.0 ** -15).all()
                if held:     # earlier tokens, rounded again where the scale grew
                    y = were[blk][:, :held] * (s_was[blk] / s_new[blk])[:, None, None]
                    err = np.abs(stored[blk][:, :held] - y)
                    assert (err <= half_step(y, fmt) * (1 + 2.0 ** -20) + 2.0 ** -15).all()
                    same = s_was[blk] == s_new[blk]
                    assert np.array_equal(stored[blk][same, :held], were[blk][same, :held])
            at += n
        # nothing else was written
        a, b_ = codes.view(torch.uint8).numpy(), cpu[c].view(torch.uint8).numpy()
        assert np.array_equal(a[~touched], b_[~touched])
        assert np.array_equal(s_new[~touched], s_was[~touched], equal_nan=True)
        # read: code * scale in fp32, rounded once
        at = 0
        for b, (s, n) in enumerate(zip(start, new)):
            for i in range(n):
                blk, slot = int(table[b, (s + i) // bt]), (s + i) % bt
                want = (codes[blk][:, slot].float() * scale[blk][:, None]).to(DTYPES[dtype])
                assert torch.equal(got[at + i].cpu(), want)
            at += n


def test_slots_after_the_tokens_keep_their_bytes(lib):
    cpu, table = filled_cache([20], 2, 64, 32, "int8", np.random.default_rng(1))
    dev = to_dev(cpu)
    x = torch.randn(4, 2, 64, device="cuda", dtype=torch.float16)
    kb.kv_write(dev, x, x, rng_of(table, [16], [4]))
    blk = int(table[0, 0])
    assert torch.equal(dev.k.cpu()[blk, :, 20:], cpu["k"][blk, :, 20:])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_special_values(lib, fmt):
    """Zeros, infinities, NaN, values under the scale floor, subnormals."""
    x = torch.zeros(32, 5, 16, dtype=torch.float32)
    x[3, 1, 2], x[4, 1, 3], x[5, 1, 4], x[6, 1, 5] = float("inf"), -float("inf"), float("nan"), 2.0
    x[:, 2] = float("nan")
    x[:, 3] = 1e-30
    x[:, 4] = 1e-41
    dev = kb.KVCache.empty(2, 5, 16, 32, dtype=CODES[fmt])
    table = torch.tensor([[1]], dtype=torch.int32)
    r = rng_of(table, [0], [32])
    kb.kv_write(dev, x.cuda(), x.cuda(), r)
    out = [torch.empty_like(x, device="cuda") for _ in "kv"]
    kb.kv_read(dev, *out, r)
    for o, scale in zip(out, (dev.k_scale, dev.v_scale)):
        o, s = o.cpu(), scale[1].cpu()
        assert torch.isfinite(o).all()
        q = QMAX[fmt]
        assert s[1] == np.float32(2.0 / q)
        assert (s[[0, 2, 3, 4]] == 2.0 ** -64).all()
        assert (o[:, [0, 2, 4]] == 0).all()
        top = np.float32(q) * s[1]
        assert o[3, 1, 2] == top and o[4, 1, 3] == -top and o[5, 1, 4] == 0 and o[6, 1, 5] == top
        assert (abs(o[:, 3] - 1e-30) <= 2.0 ** -64).all()


def test_strides_of_a_joint_buffer_and_of_a_transposed_one(lib):
    H, D, T, bt = 2, 64, 50, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    qkv = torch.randn(T, (4 + 2 * H) * D, device="cuda", generator=g).to(torch.bfloat16)
    K = qkv[:, 4 * D:(4 + H) * D].view(T, H, D)
    V = qkv[:, (4 + H) * D:].view(T, H, D)
    table = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32)
    r = rng_of(table, [0], [T])
    a, b = (kb.KVCache.empty(4, H, D, bt) for _ in range(2))
    kb.kv_write(a, K, V, r)
    kb.kv_write(b, K.contiguous(), V.transpose(0, 1).contiguous().transpose(0, 1), r)
    for x in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(a, x), getattr(b, x))
    o1, o2 = (torch.empty(T, H, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    kb.kv_read(a, o1, o2, r)
    wide = torch.zeros(T, 3 * H * D, device="cuda", dtype=torch.bfloat16)
    th = torch.zeros(H, T, D, device="cuda", dtype=torch.bfloat16)
    kb.kv_read(a, wide[:, H * D:2 * H * D].view(T, H, D), th.transpose(0, 1), r)
    assert torch.equal(wide[:, H * D:2 * H * D].reshape(T, H, D), o1)
    assert torch.equal(th.transpose(0, 1), o2)
    assert (wide[:, :H * D] == 0).all() and (wide[:, 2 * H * D:] == 0).all()


def test_token_by_token_equals_the_bounds_of_a_prompt(lib):
    """A cache grown one token at a time: every value within the steps that its
    roundings can cost (half a final step for each growth of the scale)."""
    H, D, bt, T = 2, 64, 16, 37
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(T, H, D, device="cuda", generator=g).to(torch.float16)
    dev = kb.KVCache.empty(4, H, D, bt)
    table = torch.tensor([[3, 1, 0]], dtype=torch.int32)
    growths, was = np.zeros((3, H)), np.zeros((3, H))
    for t in range(T):
        kb.kv_write(dev, x[t:t + 1], x[t:t + 1], rng_of(table, [t], [1]))
        s = dev.k_scale.cpu().numpy()[table[0].numpy()]
        growths += s > was
        was = s
    o = [torch.empty(T, H, D, device="cuda") for _ in "kv"]
    kb.kv_read(dev, *o, rng_of(table, [0], [T]))
    blk = np.arange(T) // bt
    bound = (0.5 * growths * was)[blk][:, :, None] * (1 + 1e-5)
    for y in o:
        assert (np.abs(y.cpu().numpy() - x.float().cpu().numpy()) <= bound).all()


def test_bad_block_numbers_and_lengths_are_reported_and_skipped(lib):
    H, D, bt = 1, 64, 16
    dev = kb.KVCache.empty(3, H, D, bt)
    x = torch.ones(20, H, D, device="cuda", dtype=torch.float16)
    kb.kv_device_errors(clear=True)
    kb.kv_write(dev, x, x, rng_of(torch.tensor([[1, 3]], dtype=torch.int32), [0], [20]))
    assert kb.kv_device_errors(clear=True) == {"block": True, "bounds": False, "wait": False}
    assert (dev.k[1] == 127).all() and (dev.k[0] == 0).all() and (dev.k[2] == 0).all()
    kb.kv_write(dev, x, x, rng_of(torch.tensor([[0, -1]], dtype=torch.int32), [0], [20]))
    assert kb.kv_device_errors(clear=True)["block"]
    # more tokens than the range's bounds, and than the buffer has
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 1]], **i32)
    for start, cu, most, longest in (([0], [0, 20], 19, 32), ([13], [0, 20], 20, 32),
                                     ([0], [0, 21], 21, 32), ([-1], [0, 20], 20, 32)):
        before = dev.k.clone()
        kb.kv_write(dev, x, x, kb.kv_range(table, torch.tensor(start, **i32),
                                           torch.tensor(cu, **i32), most, longest))
        assert kb.kv_device_errors(clear=True) == {"block": False, "bounds": True, "wait": False}
        assert torch.equal(dev.k, before)


def test_other_stream_and_graph(lib):
    H, D, bt = 2, 64, 32
    x = torch.randn(33, H, D, device="cuda", dtype=torch.float16)
    table = torch.tensor([[1, 0]], dtype=torch.int32)
    r = rng_of(table, [0], [33])
    ref, dev = (kb.KVCache.empty(2, H, D, bt) for _ in range(2))
    kb.kv_write(ref, x, x, r)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = [torch.empty_like(x) for _ in "kv"]
    with torch.cuda.stream(s):
        kb.kv_write(dev, x, x, r)
    s.synchronize()
    assert torch.equal(dev.k, ref.k)
    dev.k.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        kb.kv_write(dev, x, x, r)
        kb.kv_read(dev, *out, r)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(dev.k, ref.k) and torch.equal(dev.v_scale, ref.v_scale)
    # half a step, and the rounding of what is read to fp16
    assert (out[0].float() - x.float()).abs().max() <= 0.51 * ref.k_scale.max() + 2.0 ** -11 * x.abs().max()


def test_nothing_to_do(lib):
    dev = kb.KVCache.empty(1, 1, 64, 16)
    e = torch.empty(0, 1, 64, device="cuda", dtype=torch.float16)
    i32 = dict(dtype=torch.int32, device="cuda")
    kb.kv_write(dev, e, e, kb.kv_range(torch.zeros(0, 1, **i32), torch.zeros(0, **i32),
                                       torch.zeros(1, **i32), 0, 0))
    kb.kv_write(dev, e, e, kb.kv_range(torch.zeros(2, 1, **i32), torch.zeros(2, **i32),
                                       torch.zeros(3, **i32), 0, 0))
    torch.cuda.synchronize()
    assert (dev.k_scale == 0).all()
