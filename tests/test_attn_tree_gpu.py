"""Attention of trees of new tokens over the 8-bit cache against the formula in 64 bits,
and the masks that trees are given by.  Tolerances as in test_attn_kv8_gpu.py."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kernels_b200 as kb
from draft_ref import pack_bits, random_parents, tree_attention, tree_masks
from kv_ref import DTYPES, ROUND, f64, filled_cache, values

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device="cuda")


def run_case(start, new, Hq, H, D, bt, fmt, dtype, window=0, with_sinks=False, seed=0, sees=None,
             words=None, qscale=1.0):
    rng = np.random.default_rng(seed)
    lens = [s + n for s, n in zip(start, new)]
    cpu, table = filled_cache(lens, H, D, bt, fmt, rng)
    dev = kb.KVCache(*(cpu[x].cuda() for x in ("k", "v", "k_scale", "v_scale")))
    T, cu = sum(new), np.cumsum([0] + list(new))
    q = torch.from_numpy(rng.normal(0, qscale, (T, Hq, D)).astype(np.float32)).to(DTYPES[dtype])
    sinks = rng.normal(0, 2, Hq).astype(np.float32) if with_sinks else None
    words = words or -(-max(new) // 32)
    mask, pos = np.full((T, words), -1, np.int32), np.zeros(T, np.int32)
    see, first = [], []
    for b, (s, n) in enumerate(zip(start, new)):
        m, depth = tree_masks(random_parents(n, rng)) if n else (np.zeros((0, 0), bool), [])
        if sees is not None:
            m = sees(b, n, m)
        see.append(m)
        first.append([max(0, s + d - window + 1) if window else 0 for d in depth])
        bits = pack_bits(m, words)
        if n % 32:              # bits behind the tokens count for nothing
            bits[:, n // 32] |= np.int32(-1) << np.int32(n % 32)
        mask[cu[b]:cu[b + 1], :-(-n // 32)] = bits[:, :-(-n // 32)]
        pos[cu[b]:cu[b + 1]] = [s + d for d in depth]
    r = kb.kv_range(table.cuda(), torch.tensor(start, **I32), torch.tensor(cu, **I32), max(new), max(lens))
    scale = D ** -0.5
    P = kb.attn_params(Hq, DTYPES[dtype], scale=scale, window=window)
    ws = kb.AttnWorkspace(dev, r, P)
    qd = q.cuda()
    out, lse = torch.full_like(qd, float("nan")), torch.full((T, Hq), float("nan"), device="cuda")
    args = dict(positions=torch.from_numpy(pos).cuda() if window else None,
                sinks=None if sinks is None else torch.from_numpy(sinks).cuda())
    md = torch.from_numpy(mask).cuda()
    kb.kv_device_errors(clear=True)
    kb.attn_tree_kv8(dev, qd, out, r, md, P, ws, lse=lse, **args)
    assert not any(kb.kv_device_errors().values())
    for b, (s, n) in enumerate(zip(start, new)):
        if not n:
            continue
        at = slice(cu[b], cu[b + 1])
        K, V = (values(cpu, x, table, b, s + n, bt) for x in ("k", "v"))
        o, l, a, mag = tree_attention(f64(q[at]), K, V, s, np.float64(np.float32(scale)), see[b], first[b],
                                      None if sinks is None else sinks.astype(np.float64))
        d = (D + 8) * 2.0 ** -24 * mag + 2.0 ** -20
        tol = ROUND[dtype] * abs(o) * 1.01 + a * (2.0 ** -11 + 2 * d) + 1e-7
        got = f64(out[at])
        assert np.isfinite(got).all()
        worst = (abs(got - o) / tol).max()
        assert worst <= 1, f"sequence {b}: {worst} of the tolerance"
        gl = lse[at].cpu().double().numpy()
        fin = np.isfinite(l)
        assert (gl[~fin] == -np.inf).all()
        assert (abs(gl[fin] - l[fin]) <= d + 2.0 ** -20 * (1 + abs(l[fin]))).all()
    again, lse2 = torch.empty_like(out), torch.empty_like(lse)
    kb.attn_tree_kv8(dev, qd, again, r, md, P, ws, lse=lse2, **args)
    assert torch.equal(again, out) and torch.equal(lse2, lse)
    return dev, qd, out, lse, r, P, ws, args


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads", [(8, 8, 64), (8, 4, 128), (1, 1, 16), (4, 2, 96), (3, 3, 256), (2, 2, 80)])
def test_few_rows(lib, heads, dtype, fmt):
    Hq, H, D = heads
    n = 4 if D <= 128 else 3
    run_case([0, 1, 15, 16, 63, 200, 701], [n, 1, n, 2, n, 0, n], Hq, H, D, 16, fmt, dtype, 0, True)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("n", [5, 20, 32])
def test_up_to_a_word_of_few_rows(lib, n, fmt):
    run_case([0, 27, 333], [n, 1, n - 2], 2, 2, 64, 32, fmt, "f16", 0, False, seed=n)
    run_case([0, 27, 333], [n, 1, n - 2], 2, 2, 64, 16, fmt, "bf16", 25, True, seed=n)


@pytest.mark.parametrize("shape", [
    # start, new, q heads, heads, dim
    ([0], [9], 64, 8, 64), ([777], [7], 64, 8, 64), ([300, 0, 5], [17, 0, 33], 20, 4, 64),
    ([1000, 31], [65, 64], 16, 2, 64), ([0, 700], [129, 64], 8, 1, 128), ([64], [200], 3, 1, 96),
    ([31, 9], [16, 257], 5, 1, 256), ([2], [9], 32, 1, 48), ([90, 127, 128, 129], [31, 32, 33, 1], 16, 2, 64),
    ([50], [700], 4, 1, 64), ([513] * 12, [8] * 12, 32, 8, 128), ([4000], [24], 64, 8, 64)])
@pytest.mark.parametrize("window,sinks", [(0, False), (50, True)])
def test_many_rows(lib, shape, window, sinks):
    start, new, Hq, H, D = shape
    run_case(start, new, Hq, H, D, 32, "int8", "bf16", window, sinks, seed=5)
    run_case(start, new, Hq, H, D, 16, "e4m3", "f16", window, sinks, seed=6)


@pytest.mark.parametrize("group", [1, 8])
def test_any_mask(lib, group):
    """Masks of no tree: later tokens, no own key, nothing at all."""
    rng = np.random.default_rng(1)

    def sees(b, n, m):
        m = rng.random((n, n)) < 0.4
        m[::3] = False
        return m
    for start, new in (([0, 3], [4, 3]), ([0, 16, 200], [30, 40, 64]), ([0], [300])):
        for sinks in (False, True):
            run_case(start, new, 2 * group, 2, 64, 16, "int8", "f16", 0, sinks, seed=2, sees=sees, words=11)
            run_case(start, new, 2 * group, 2, 128, 32, "e4m3", "bf16", 0, sinks, seed=3, sees=sees)


def test_empty_rows_give_zeros(lib):
    *_, out, lse, r, P, ws, args = run_case([0], [20], 8, 1, 64, 16, "e4m3", "f16",
                                            sees=lambda b, n, m: np.zeros((n, n), bool))
    assert not out.any() and (lse == -float("inf")).all()
    *_, out, lse, r, P, ws, args = run_case([0], [3], 8, 1, 64, 16, "int8", "f16",
                                            sees=lambda b, n, m: np.zeros((n, n), bool))
    assert not out.any() and (lse == -float("inf")).all()


@pytest.mark.parametrize("n", [2, 30])
def test_a_chain_is_the_causal_call(lib, n):
    """A chain's masks give what attn_kv8 gives, to the roundings of both."""
    dev, q, _, _, r, P, ws, args = run_case([100, 40], [n, n], 8, 2, 64, 16, "int8", "f16", 37, True)
    T = 2 * n
    par = torch.arange(-1, n - 1, **I32).repeat(2)
    mask, pos = torch.full((T, 3), -1, **I32), torch.empty(T, **I32)
    kb.draft_tree(par, r, mask, pos, window=37)
    out, want = torch.empty_like(q), torch.empty_like(q)
    kb.attn_tree_kv8(dev, q, out, r, mask, P, ws, positions=pos, sinks=args["sinks"])
    kb.attn_kv8(dev, q, want, r, P, ws, sinks=args["sinks"])
    assert (out.float() - want.float()).abs().max() <= 2 * 2.0 ** -11 * 4 * want.abs().max().float()
    assert pos.tolist() == list(range(100, 100 + n)) + list(range(40, 40 + n))


def test_long_context(lib):
    run_case([30001], [4], 16, 2, 64, 64, "int8", "f16", 0, True, seed=1, qscale=2.0)
    run_case([20000, 7], [40, 3], 16, 2, 64, 64, "e4m3", "bf16", 0, False, seed=2, qscale=2.0)
    run_case([30000], [20], 16, 1, 128, 128, "int8", "bf16", 4000, True, seed=3, qscale=2.0)


@pytest.mark.parametrize("window", [0, 1, 3, 100])
def test_masks_from_parents(lib, window):
    rng = np.random.default_rng(7)
    new, start = [1, 0, 33, 64, 5, 300, 1], [0, 3, 77, 1, 2, 100000, 9]
    cu = np.cumsum([0] + new)
    T, words = sum(new), 12
    parents = np.zeros(T, np.int32)
    want, pos = np.zeros((T, words), np.int32), np.zeros(T, np.int32)
    for b, n in enumerate(new):
        p = random_parents(n, rng) if n else []
        if n > 30:
            p[7], p[9], p[11] = -1, 9, 1 << 30      # a second root; nothing that comes before
        parents[cu[b]:cu[b + 1]] = p
        if n:
            see, depth = tree_masks(p, window)
            want[cu[b]:cu[b + 1]], pos[cu[b]:cu[b + 1]] = pack_bits(see, words), np.array(depth) + start[b]
    r = kb.kv_range(torch.zeros(len(new), 1 << 16, **I32), torch.tensor(start, **I32),
                    torch.tensor(cu, **I32), 384, 1 << 20)
    mask = torch.full((T + 2, words + 3), 5, **I32)
    where = torch.full((T + 2,), 5, **I32)
    kb.draft_tree(torch.from_numpy(parents).cuda(), r, mask[:T, 1:words + 1], where[:T], window=window)
    assert not any(kb.kv_device_errors().values())
    assert np.array_equal(mask[:T, 1:words + 1].cpu().numpy(), want)
    assert np.array_equal(where[:T].cpu().numpy(), pos)
    assert (mask[T:] == 5).all() and (mask[:, 0] == 5).all() and (mask[:, words + 1:] == 5).all()
    assert (where[T:] == 5).all()


def test_captured_masks(lib):
    """Masks, positions and lengths follow the device's memory in a replay."""
    dev, q, out, lse, r, P, ws, args = run_case([100, 40], [20, 20], 8, 2, 64, 16, "int8", "f16", 37, True)
    par = torch.arange(-1, 19, **I32).repeat(2)
    mask, pos = torch.zeros(40, 1, **I32), torch.zeros(40, **I32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        kb.draft_tree(par, r, mask, pos, window=37)
        kb.attn_tree_kv8(dev, q, out, r, mask, P, ws, positions=pos, sinks=args["sinks"], lse=lse)
    par.copy_(torch.tensor(random_parents(20, np.random.default_rng(4)) * 2, **I32))
    g.replay()
    want, wl = torch.empty_like(out), torch.empty_like(lse)
    m2, p2 = torch.zeros_like(mask), torch.zeros_like(pos)
    kb.draft_tree(par, r, m2, p2, window=37)
    kb.attn_tree_kv8(dev, q, want, r, m2, P, ws, positions=p2, sinks=args["sinks"], lse=wl)
    torch.cuda.synchronize()
    assert torch.equal(m2, mask) and torch.equal(want, out) and torch.equal(wl, lse)


# (few rows in registers, in shared memory; rows as columns, one and both groups; many rows; 256 dims)
FORMS = [([90, 40], [2, 2], 8, 2, 64), ([90, 40], [6, 3], 8, 2, 64), ([300, 40], [5, 8], 8, 2, 128),
         ([300, 700], [16, 13], 8, 2, 64), ([300, 700], [30, 13], 8, 2, 64), ([90, 40], [7, 8], 4, 2, 256)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_a_bad_query_spoils_its_own_row_only(lib, form, dtype):
    """The other rows' references may move with the spoilt row's, so both runs lie within run_case's
    tolerance of the formula; codes times scales are at most 2 here, and so |o| and sum p |v|."""
    dev, q, out, lse, r, P, ws, _ = run_case(*form, 16, "int8", dtype, 0, False, seed=9)
    T = q.shape[0]
    mask = torch.full((T, 1), -1, **I32)      # everything
    good = torch.empty_like(out)
    kb.attn_tree_kv8(dev, q, good, r, mask, P, ws)
    D = q.shape[2]
    d = (D + 8) * 2.0 ** -24 * float(q.float().abs().sum(2).max()) * 2 * D ** -0.5 + 2.0 ** -20
    tol = 2 * (ROUND[dtype] * 2 * 1.01 + 2 * (2.0 ** -11 + 2 * d) + 1e-7)
    for bad in (float("nan"), float("inf"), -float("inf")):
        spoilt = q.clone()
        spoilt[1, 3, 5] = bad
        got = torch.empty_like(out)
        kb.attn_tree_kv8(dev, spoilt, got, r, mask, P, ws)
        others = torch.ones(T, q.shape[1], dtype=torch.bool, device="cuda")
        others[1, 3] = False
        a, b = got[others].float(), good[others].float()
        assert (a - b).abs().max() <= tol
        if bad != bad:
            assert got[1, 3].isnan().all()
    assert not any(kb.kv_device_errors().values())


@pytest.mark.parametrize("form", FORMS)
def test_strides_and_what_lies_around(lib, form):
    """Queries in the middle of wider rows, masks with other words around them, and output that is
    nobody's."""
    dev, q, _, _, r, P, ws, _ = run_case(*form, 16, "e4m3", "f16", 0, False, seed=11)
    T, Hq, D = q.shape
    rng = np.random.default_rng(11)
    wide = torch.full((T, Hq + 3, D + 16), float("nan"), device="cuda").half()
    wide[:, 1:Hq + 1, 8:D + 8] = q
    out = torch.full((T + 2, Hq + 1, D + 8), 7.0, device="cuda").half()
    mask = torch.full((T, 5), -1, **I32)
    mask[:, 2] = torch.from_numpy(rng.integers(0, 1 << 30, T).astype(np.int32)).cuda()
    dense = torch.empty_like(q)
    kb.attn_tree_kv8(dev, q, dense, r, mask[:, 2:3].contiguous(), P, ws)
    kb.attn_tree_kv8(dev, wide[:, 1:Hq + 1, 8:D + 8], out[:T, :Hq, :D], r, mask[:, 2:3], P, ws)
    assert torch.equal(out[:T, :Hq, :D], dense) and torch.isfinite(dense).all()
    assert (out[T:] == 7).all() and (out[:, Hq:] == 7).all() and (out[:, :, D:] == 7).all()


@pytest.mark.parametrize("new", [2, 5, 9])
def test_more_sequences_than_threads(lib, new):
    run_case([i % 37 for i in range(1100)], [new if i % 3 else 1 for i in range(1100)], 8, 1, 64, 16, "int8",
             "f16", 0, False, seed=3)
    run_case([i % 37 for i in range(500)], [0 if i % 5 else new for i in range(500)], 8, 1, 128, 16, "e4m3",
             "bf16", 9, True, seed=3)


@pytest.mark.parametrize("form", FORMS)
def test_sharp_and_flat_scores(lib, form):
    for qscale in (0.0, 40.0):
        run_case(*form, 32, "int8", "f16", 0, True, seed=13, qscale=qscale)
        run_case(*form, 32, "e4m3", "bf16", 20, False, seed=13, qscale=qscale)
