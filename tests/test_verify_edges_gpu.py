"""Verification of drafted tokens where the definition is decided by one token among many: ties,
rows at odd addresses, masked tokens, random numbers at the ends and next to borders."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from kv_ref import DTYPES, f64
from test_verify_gpu import call

pytestmark = pytest.mark.gpu


def rows_at_odd_places(z, dtype, gap):
    """z [rows, V] on the GPU with `gap` elements before and between its rows."""
    n, V = z.shape
    flat = torch.zeros(n * (V + gap) + 16, dtype=DTYPES[dtype], device="cuda")
    view = flat[gap:gap + n * (V + gap)].view(n, V + gap)[:, :V]
    view.copy_(torch.from_numpy(z).to(DTYPES[dtype]))
    return view


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("V", [1, 5, 9, 1001, 50021])
@pytest.mark.parametrize("gap", [0, 1, 2, 3])
def test_greedy_ties_at_every_offset(lib, V, gap, dtype):
    """The first of equal largest logits, in rows that begin and end inside a 16-byte chunk: the
    root's row decides about its child, the child's about what follows."""
    rng = np.random.default_rng(V + gap)
    n = 48                                    # sequences: a root and its child
    z = rng.normal(0, 1, (2 * n, V)).astype(np.float32)
    for r in range(2 * n):
        if r % 6 == 5:
            z[r] = 1.0                        # all are equal
            continue
        # one of the first tokens and some of the others: of the next chunks, far behind, the last
        ties = {r % 7, 8 + r % 9, 1024 + r % 8, 4096 + r % 16, int(rng.integers(V)), V - 1 - r % 3}
        z[r, [t for t in sorted(ties)[r % 2:] if 0 <= t < V]] = 7.0
    first = z.argmax(1)                       # (numpy: the first)
    view = rows_at_odd_places(z, dtype, gap)
    assert (f64(view).argmax(1) == first).all()
    tokens = np.zeros(2 * n, np.int64)
    tokens[1::2] = first[0::2]
    cu = list(range(0, 2 * n + 1, 2))
    count, path, nxt = call(view, tokens, cu, None)
    assert count == [2] * n and path == list(range(2 * n)) and nxt == first[1::2].tolist()
    # a later one of the equals is refused, and what follows is the first
    later = [np.nonzero(z[r] == z[r].max())[0] for r in range(0, 2 * n, 2)]
    tokens[1::2] = [t[-1] if len(t) > 1 else V + 1 for t in later]
    count, _, nxt = call(view, tokens, cu, None)
    assert count == [1] * n and nxt == first[0::2].tolist()


def first_possible(kind, B, V, masked, dtype):
    """B sequences, the same root's row: `masked` tokens that cannot come lie before all that can, but for
    (kind "chosen") one among them, which is rejected.  Rejections leave the smallest token behind them
    with something; the random number 0 has to find it."""
    n = {"chosen": 2, "once": 2, "often": 4}[kind]
    z = np.full(V, -np.inf, np.float32)
    z[masked::997] = 0.0                             # few for the target, many for the draft, so that the
    q = np.random.default_rng(V).normal(0, 1, V).astype(np.float32)   # target's sum is the smaller one
    q[:masked] = -np.inf
    drawn = np.argsort(-np.where(z == 0, -np.inf, q))[:n - 1]         # likely ones that cannot come
    if kind == "chosen":
        z[masked // 2] = 3.0
        drawn = np.array([masked // 2])
    u = np.full((B, n), 0.999, np.float32)
    tokens = np.concatenate([[0], drawn])
    parents = np.array([-1] + [0] * (n - 1)) if kind == "often" else None
    rows = torch.from_numpy(np.stack([z] + [np.zeros(V, np.float32)] * (n - 1)))
    rows = rows.to(DTYPES[dtype]).cuda().repeat(B, 1)
    guess = None if kind == "chosen" else torch.from_numpy(q).to(DTYPES[dtype]).cuda().expand(n, V).repeat(B, 1)
    cu = [n * b for b in range(B + 1)]
    return rows, np.tile(tokens, B), cu, None if parents is None else np.tile(parents, B), guess, u.reshape(-1)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("B,V,masked", [(128, 128256, 8192), (128, 128256, 100001), (200, 33000, 20000)])
@pytest.mark.parametrize("kind", ["chosen", "once", "often"])
def test_masked_tokens_are_never_what_follows(lib, kind, B, V, masked, dtype):
    """Thousands of tokens that cannot come are together still none: for the random number 0 `next` is the
    first token that can."""
    rows, tokens, cu, parents, guess, u = first_possible(kind, B, V, masked, dtype)
    n = cu[1]
    from draft_ref import verify
    par = [-1] + [0] * (n - 1) if parents is not None else list(range(-1, n - 1))
    path, nxt, _ = verify(f64(rows[:n]), tokens[:n], par, 1.0, None if guess is None else f64(guess[:n]),
                          1.0, u[:n], 0.0)
    assert path == [0] and nxt == masked
    got = call(rows, tokens, cu, parents, draft=guess, uniform=u, last=np.zeros(B, np.float32))
    assert got[0] == [1] * B and got[2] == [nxt] * B


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_lowest_finite_logits_are_tokens(lib, dtype):
    """A row of the type's lowest value, as a mask leaves it, beside tokens that cannot come: only the former
    can, each as often as the others."""
    low, V = float(np.finfo(np.float16 if dtype == "f16" else np.float32).min), 1000
    z = torch.full((40, V), float("-inf"))
    z[:, 300:310] = low
    z = z.to(DTYPES[dtype]).cuda()
    last = (np.arange(40, dtype=np.float32) + 0.5) / 40
    want = [300 + b // 4 for b in range(40)]
    assert call(z, np.zeros(40, np.int64), list(range(41)), None, uniform=np.zeros(40, np.float32),
                last=last)[2] == want
    # .. also behind a child that was rejected, and whose token is one of them
    z2 = z.repeat_interleave(2, 0)
    got = call(z2, np.tile([0, 304], 40), [2 * b for b in range(41)], None,
               uniform=np.tile(np.float32([0, 0.5]), 40), last=(np.arange(40, dtype=np.float32) + 0.5) / 40)
    left = [t for t in range(300, 310) if t != 304]
    assert got[0] == [1] * 40 and got[2] == [left[int(x * 9)] for x in last]


def softmax_rows(z, scale):
    z = z * np.float64(np.float32(scale))
    e = np.exp(z - z.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True)


# Random numbers lie 2^-9 to 2^-21 to either side of a border.  They are fp32, rounded to 2^-25 at
# most where they are below 1/2 and a border of at least 1/8 moves them by 2^-22 of it; what side they
# are on is worked out from the rounded ones, in fp64, whose sums are right to 2^-45 of the little that is left.
SIDES = np.array([s * 2.0 ** -k for k in range(9, 22) for s in (-1, 1)])


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("V,top,scale", [(4099, 0.99, 1.3), (4099, 0.5, 0.7), (20011, 0.998, 1.0)])
def test_second_children_near_their_border(lib, V, top, scale, dtype):
    """A looked-up child that has most of the probability is rejected; whether the next is accepted against
    what is left is decided as 64-bit sums do."""
    rng = np.random.default_rng(V)
    B = 26 * (40 if V < 9000 else 10)
    z = torch.from_numpy(rng.normal(0, 1, (3 * B, V)).astype(np.float32)).to(DTYPES[dtype])
    root = z[::3].double().numpy()
    rest = np.log(np.exp(root * scale).sum(1))
    root[:, 7] = (rest + np.log(top / (1 - top))) / scale      # p about `top`,
    root[:, V - 9] = (rest + np.log(0.45)) / scale             # and a third of what is left without it
    z[::3] = torch.from_numpy(root).to(z.dtype)
    p = softmax_rows(f64(z[::3]), scale)
    r, R = p[:, V - 9], p.sum(1) - p[:, 7]
    u = np.full((B, 3), 0.9999, np.float32)
    u[:, 2] = (r / R * (1 + np.resize(SIDES, B))).astype(np.float32)
    assert (u[:, 1] > p[:, 7]).all() and (0.125 < u[:, 2]).all() and (u[:, 2] < 0.5).all()
    want = (u[:, 2].astype(np.float64) * R < r)
    assert 0.4 < want.mean() < 0.6
    tokens, parents = np.tile([0, 7, V - 9], B), np.tile([-1, 0, 0], B)
    count, path, _ = call(z.cuda(), tokens, [3 * b for b in range(B + 1)], parents, scale=scale,
                          uniform=u.reshape(-1), last=np.full(B, 0.5, np.float32))
    assert (np.array(count) == 1 + want).all()
    assert (np.array(path).reshape(B, 3)[:, 1] == np.where(want, 3 * np.arange(B) + 2, -1)).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("V,scale", [(4099, 1.3), (20011, 0.7)])
def test_first_children_near_their_border(lib, V, scale, drawn, dtype):
    """.. and so is a first child, of the draft's distribution or looked up."""
    rng = np.random.default_rng(V + 1)
    B = 26 * (40 if V < 9000 else 10)
    z = torch.from_numpy(rng.normal(0, 2, (2 * B, V)).astype(np.float32)).to(DTYPES[dtype])
    z[:, 5] = 4.0 + np.log(V) / scale
    d = torch.from_numpy(rng.normal(0, 2, (2 * B, V)).astype(np.float32)).to(DTYPES[dtype])
    d[:, 5] = 6.0 + np.log(V) / scale
    p = softmax_rows(f64(z[::2]), scale)[:, 5]
    q = softmax_rows(f64(d[::2]), scale)[:, 5] if drawn else np.ones(B)
    u = np.full((B, 2), 0.5, np.float32)
    u[:, 1] = (p / q * (1 + np.resize(SIDES, B))).astype(np.float32)
    assert (0.125 < u[:, 1]).all() and (u[:, 1] < 1).all()     # (rounded by 2^-25: 2^-22 of 1/8)
    want = u[:, 1].astype(np.float64) * q < p
    assert 0.4 < want.mean() < 0.6
    count, _, _ = call(z.cuda(), np.tile([0, 5], B), [2 * b for b in range(B + 1)], None, scale=scale,
                       draft=d.cuda() if drawn else None, draft_scale=scale, uniform=u.reshape(-1),
                       last=np.full(B, 0.5, np.float32))
    assert (np.array(count) == 1 + want).all()
