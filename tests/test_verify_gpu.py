"""Verification of drafted tokens against the definition in 64 bits.  Counts, paths and
tokens have to be equal; inputs whose random numbers lie within 2^-18 of an acceptance's
border (the sums behind it are fp32) are drawn again beforehand."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import kernels_b200 as kb
from draft_ref import random_parents, verify
from kv_ref import DTYPES, f64

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device="cuda")


def call(z, tokens, cu, parents, scale=1.0, draft=None, draft_scale=1.0, uniform=None, last=None, longest=None):
    B, (T, V) = len(cu) - 1, z.shape
    P = kb.verify_params(B, T, longest or max(np.diff(cu)), V, z.dtype, scale=scale, draft_scale=draft_scale)
    ws = kb.VerifyWorkspace(P)
    ws.buffer.fill_(0xFF)                 # any content
    count, nxt = (torch.full((B,), 77, **I32) for _ in range(2))
    path = torch.full((T,), 77, **I32)

    def dev(x, t):
        return None if x is None else torch.as_tensor(np.asarray(x)).to(t).cuda()
    a = dict(draft=draft, parents=dev(parents, torch.int32), uniform=dev(uniform, torch.float32),
             uniform_next=dev(last, torch.float32))
    kb.verify_drafts(z, dev(tokens, torch.int32), dev(cu, torch.int32), count, path, nxt, P, ws, **a)
    c, p, n = count.tolist(), path.tolist(), nxt.tolist()
    kb.verify_drafts(z, dev(tokens, torch.int32), dev(cu, torch.int32), count, path, nxt, P, ws, **a)
    assert (c, p, n) == (count.tolist(), path.tolist(), nxt.tolist())
    return c, p, n


def expected(z, tokens, cu, parents, scale, draft, draft_scale, uniform, last):
    zz, dd = f64(z), None if draft is None else f64(draft)
    count, path, nxt, near = [], [77] * len(z), [], []
    for b in range(len(cu) - 1):
        at = slice(cu[b], cu[b + 1])
        n = cu[b + 1] - cu[b]
        if n == 0:
            count.append(0), nxt.append(-1), near.append(np.inf)
            continue
        par = list(range(-1, n - 1)) if parents is None else list(parents[at])
        got, t, close = verify(zz[at], tokens[at], par, np.float64(np.float32(scale)),
                               None if dd is None else dd[at], np.float64(np.float32(draft_scale)),
                               None if uniform is None else uniform[at], None if last is None else last[b])
        count.append(len(got)), nxt.append(t), near.append(close)
        path[at] = [cu[b] + i for i in got] + [-1] * (n - len(got))
    return count, path, nxt, near


def make(new, V, dtype, seed, trees=True, drawn=True, masked=0.0, noise=0.7, wide=3):
    rng = np.random.default_rng(seed)
    T, cu = sum(new), np.cumsum([0] + list(new))
    z = rng.normal(0, 3, (T, V)).astype(np.float32)
    if masked:
        z[rng.random((T, V)) < masked] = -np.inf
    guess = z + noise * rng.normal(0, 1, (T, V)).astype(np.float32)
    parents = np.concatenate([random_parents(n, rng, wide) for n in new if n]) if trees else None
    tokens = np.zeros(T, np.int64)
    order = np.argsort(-guess, axis=1)
    for b, n in enumerate(new):
        for i in range(1, n):
            p = parents[cu[b] + i] if trees else i - 1
            row = guess[cu[b] + p]
            if drawn:
                w = np.exp(row.astype(np.float64) - row.max())
                tokens[cu[b] + i] = rng.choice(V, p=w / w.sum())
            else:
                tokens[cu[b] + i] = order[cu[b] + p, i % min(4, V)]
    u, last = rng.random(T).astype(np.float32), rng.random(len(new)).astype(np.float32)
    t = DTYPES[dtype]
    return (torch.from_numpy(z).to(t).cuda(), tokens, cu, parents,
            torch.from_numpy(guess).to(t).cuda() if drawn else None, u, last)


def check(new, V, dtype, seed, scale=1.0, draft_scale=1.0, **kw):
    z, tokens, cu, parents, draft, u, last = make(new, V, dtype, seed, **kw)
    rng = np.random.default_rng(seed + 1000)
    for _ in range(20):
        want = expected(z, tokens, cu, parents, scale, draft, draft_scale, u, last)
        close = [b for b, x in enumerate(want[3]) if x < 2.0 ** -18]
        if not close:
            break
        for b in close:
            u[cu[b]:cu[b + 1]], last[b] = rng.random(new[b]), rng.random()
    got = call(z, tokens, cu, parents, scale, draft, draft_scale, u, last)
    assert got == want[:3]
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("V", [1, 2, 31, 1000, 4099, 50021])
@pytest.mark.parametrize("drawn", [True, False])
def test_chains(lib, V, drawn, dtype):
    check([1, 2, 6, 0, 5, 9], V, dtype, V, trees=False, drawn=drawn)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("V", [7, 257, 5003, 33000])
@pytest.mark.parametrize("drawn", [True, False])
def test_trees(lib, V, drawn, dtype):
    check([1, 12, 31, 0, 5, 64, 2], V, dtype, V, drawn=drawn)
    check([40, 3], V, dtype, V + 1, drawn=drawn, wide=20, scale=0.7, draft_scale=1.3)


@pytest.mark.parametrize("drawn", [True, False])
def test_masked_and_large(lib, drawn):
    check([8, 20], 128256, "f16", 0, drawn=drawn, masked=0.9)
    check([6] * 4, 201088, "bf16", 1, drawn=drawn, trees=False, scale=1.25, draft_scale=1.25)


def test_many_sequences(lib):
    got = check([1 + i % 7 for i in range(300)], 300, "f16", 3, trees=False)
    assert len(set(got[0])) > 3
    check([1 + i % 9 for i in range(200)], 300, "f32", 4, drawn=False)


def test_longest_trees(lib):
    rng = np.random.default_rng(0)
    z, tokens, cu, parents, draft, u, last = make([1024, 3], 64, "f32", 5, drawn=False)
    parents[1:1024] = 0           # all are the root's children, tokens many times over
    tokens[1:1024] = rng.integers(0, 64, 1023)
    want = expected(z, tokens, cu, parents, 1.0, None, 1.0, u, last)
    assert min(want[3]) > 2.0 ** -18
    assert call(z, tokens, cu, parents, 1.0, None, 1.0, u, last) == want[:3]
    check([1024], 40, "f32", 6, trees=False, drawn=False)


@pytest.mark.parametrize("took", [None, 1, 400, 1022])
@pytest.mark.parametrize("slope", [0.02, 0.6])
def test_many_siblings(lib, slope, took):
    """A root with 1023 children, the likeliest tokens first, that are rejected one after the
    other (but one): what is left of p falls to e^-20 and e^-614."""
    n, V = 1024, 20011
    z = torch.full((n, V), -math.inf, device="cuda")
    order = torch.from_numpy(np.random.default_rng(1).permutation(V)[:1200])
    z[0, order.cuda()] = (-slope * torch.arange(1200.0)).cuda()
    z[1:, :7] = 0.0
    tokens = np.concatenate([[0], order[:n - 1].numpy()])
    u = np.full(n, 0.9, np.float32)
    if took:
        u[took] = 0.001
    cu, parents = [0, n], np.array([-1] + [0] * (n - 1))
    last = np.array([0.3], np.float32)
    want = expected(z, tokens, cu, parents, 1.0, None, 1.0, u, last)
    assert min(want[3]) > 2.0 ** -18 and want[0] == [2 if took else 1]
    assert call(z, tokens, cu, parents, uniform=u, last=last) == want[:3]


def test_no_tokens(lib):
    z = torch.zeros(0, 50, device="cuda")
    for u in (None, []):
        got = call(z, [], [0, 0, 0], None, uniform=u, last=None if u is None else [0.5, 0.5], longest=3)
        assert got == ([0, 0], [], [-1, -1])


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("V", [3, 1000, 50021])
def test_greedy(lib, V, dtype):
    z, tokens, cu, parents, _, _, _ = make([1, 12, 31, 0, 5, 64, 2], V, dtype, V, drawn=False, noise=0.2)
    got = call(z, tokens, cu, parents)
    assert got == expected(z, tokens, cu, parents, 1.0, None, 1.0, None, None)[:3]
    assert max(got[0]) > 1


def test_greedy_ties_go_to_the_first(lib):
    z = torch.zeros(3, 70000, device="cuda").half()
    z[:, 11] = z[:, 69999] = z[:, 40000] = 2
    z[2] = -0.0
    z[2, 5:] = 0.0
    assert call(z, [0, 11, 11], [0, 3], None) == ([3], [0, 1, 2], [0])
    assert call(z, [0, 40000, 11], [0, 3], None) == ([1], [0, -1, -1], [11])


def test_next_follows_the_distribution(lib):
    """Random numbers over a grid: each token comes as often as its probability says, to the
    grid's step, whether it is a draft's or not."""
    V, N = 5, 4000
    p = torch.tensor([0.1, 0.0, 0.4, 0.3, 0.2], dtype=torch.float64)
    q = torch.tensor([0.3, 0.1, 0.1, 0.5, 0.0], dtype=torch.float64)
    g = np.random.default_rng(0)
    tok = g.choice(V, N, p=q.numpy())
    z, d = p.log().float().cuda().repeat(2 * N, 1), q.log().float().cuda().repeat(2 * N, 1)
    tokens = np.zeros(2 * N, np.int64)
    tokens[1::2] = tok
    count, path, nxt = call(z, tokens, list(range(0, 2 * N + 1, 2)), None, draft=d,
                            uniform=g.random(2 * N), last=g.random(N))
    first = np.where(np.array(count) == 2, tok, nxt)
    got = np.bincount(first, minlength=V) / N
    # 5 standard deviations of a share of 4000
    assert (abs(got - p.numpy()) <= 5 * np.sqrt(p.numpy() * (1 - p.numpy()) / N) + 1e-12).all()


def test_ends_of_the_unit_interval(lib):
    z = torch.tensor([[-math.inf, 1.0, 0.0, 2.0, -math.inf]] * 4, device="cuda")
    for u, want in ((0.0, 1), (0.999999, 3), (1.0, 3), (5.0, 3), (-1.0, 1)):
        assert call(z[:1], [0], [0, 1], None, uniform=[0.5], last=[u])[2] == [want]
    # u = 0 takes every token that can come, u = 1 none unless it is certain; one that cannot come never
    assert call(z[:2], [0, 2], [0, 2], None, uniform=[0, 0], last=[0.5])[0] == [2]
    assert call(z[:2], [0, 0], [0, 2], None, uniform=[0, 0], last=[0.5])[0] == [1]
    assert call(z[:2], [0, 2], [0, 2], None, uniform=[0, 1], last=[0.0])[::2] == ([1], [1])


def test_rows_without_a_distribution(lib):
    good = torch.tensor([0.0, 1.0, 2.0, 0.5])
    for bad in ([math.nan, 0, 0, 0], [math.inf, 0, 0, 0], [-math.inf] * 4):
        z = good.repeat(3, 1)
        z[1] = torch.tensor(bad)
        # the child before is accepted, the one behind never; nothing follows
        args = dict(uniform=[0, 0, 0], last=[0.5])
        assert call(z.cuda(), [0, 2, 2], [0, 3], None, **args) == ([2], [0, 1, -1], [-1])
        assert call(z.cuda(), [0, 2, 2], [0, 3], None) == ([2], [0, 1, -1], [-1])
        # as a leaf
        assert call(z[:2].cuda(), [0, 2], [0, 2], None, uniform=[0, 0], last=[0.5]) == ([2], [0, 1], [-1])
        assert call(z[:2].cuda(), [0, 2], [0, 2], None) == ([2], [0, 1], [-1])
        # such a row of the draft: its children are passed over, next is drawn from p
        want = call(good.repeat(1, 1).cuda(), [0], [0, 1], None, uniform=[0], last=[0.7])[2]
        d = good.repeat(3, 1)
        d[0] = torch.tensor(bad)
        got = call(good.repeat(3, 1).cuda(), [0, 2, 2], [0, 3], None, draft=d.cuda(), uniform=[0, 0, 0], last=[0.7])
        assert got == ([1], [0, -1, -1], want)


def test_tokens_and_parents_that_are_none(lib):
    z = torch.tensor([[0.0, 1.0, 2.0, 0.5]] * 6, device="cuda")
    # tokens outside the vocabulary; a parent that is the token itself, later, or far off
    got = call(z, [0, -1, 4, 2, 2, 2], [0, 6], [-1, 0, 0, 3, 5, 1 << 20], uniform=[0.0] * 6, last=[0.999])
    assert got == ([1], [0] + [-1] * 5, [3])
    got = call(z, [0, -1, 4, 2, 2, 2], [0, 6], [-1, 0, 0, 0, 5, 3], uniform=[0.0] * 6, last=[0.0])
    assert got == ([3], [0, 3, 5, -1, -1, -1], [0])


def test_nothing_left_is_p_again(lib):
    """q = p: a rejection (random number 1) leaves nothing; the draw is from p."""
    z = torch.tensor([[0.0, -math.inf, -math.inf]] * 2, device="cuda")
    assert call(z, [0, 0], [0, 2], None, draft=z, uniform=[0, 1], last=[0.5])[2] == [0]
    assert call(z, [0, 0], [0, 2], None, uniform=[0, 1], last=[0.5])[2] == [0]
    z = torch.zeros(4, 8, device="cuda")
    got = call(z, [0, 3, 3, 4], [0, 4], [-1, 0, 0, 0], draft=z, uniform=[0, 1, 1, 0.5], last=[0.5])
    assert got[0] == [2] and got[1] == [0, 3, -1, -1]


def test_little_left(lib):
    """Siblings that take all but 2^-30 of the probability: sums in 64 bits decide."""
    z = torch.full((4, 1000), -30.0, device="cuda")
    z[0, 7], z[0, 8] = 3.0, 2.0
    parents, tokens = [-1, 0, 0, 0], [0, 7, 8, 500]
    for u, last in ((0.0005, 0.3), (0.5, 0.3), (0.0005, 0.99)):
        u = [0, 0.9999999, 0.9999999, u]
        cu = [0, 4]
        want = expected(z, np.array(tokens), cu, np.array(parents), 1.0, None, 1.0, np.array(u, np.float32),
                        np.array([last], np.float32))
        if want[3][0] > 2.0 ** -18:
            assert call(z, tokens, cu, parents, uniform=u, last=[last]) == want[:3]


def test_strides_and_bad_lengths(lib):
    z, tokens, cu, parents, draft, u, last = make([6, 3], 999, "f16", 9, trees=False)
    wide = torch.zeros(9, 1500, device="cuda").half()
    wide[:, 3:1002] = z
    other = torch.zeros(9, 1007, device="cuda").half()
    other[:, 1:1000] = draft
    want = call(z, tokens, cu, None, draft=draft, uniform=u, last=last)
    assert call(wide[:, 3:1002], tokens, cu, None, draft=other[:, 1:1000], uniform=u, last=last) == want
    # more tokens than the host said, or than there are rows; rows behind stay as they are
    got = call(z, tokens, [0, 6, 9], None, draft=draft, uniform=u, last=last, longest=4)
    assert got[0][0] == 0 and got[2][0] == -1 and got[0][1] == want[0][1] and got[1][:6] == [77] * 6
    got = call(z, tokens, [0, 6, 10], None, draft=draft, uniform=u, last=last, longest=6)
    assert got[0] == [want[0][0], 0] and got[1][6:] == [77] * 3
    got = call(z, tokens, [0, 6, 6], None, draft=draft, uniform=u, last=last, longest=6)
    assert got[0] == [want[0][0], 0] and got[1][6:] == [77] * 3
    got = call(z, tokens, [-1, 5, 9], None, draft=draft, uniform=u, last=last, longest=6)
    assert got[0][0] == 0 and got[2][0] == -1


def test_captured(lib):
    z, tokens, cu, _, draft, u, last = make([6, 3], 5000, "f16", 11, trees=False)
    P = kb.verify_params(2, 9, 6, 5000, z.dtype)
    ws = kb.VerifyWorkspace(P)
    t, c = torch.from_numpy(tokens).int().cuda(), torch.tensor(cu, **I32)
    u, last = torch.from_numpy(u).cuda(), torch.from_numpy(last).cuda()
    out = [torch.zeros(n, **I32) for n in (2, 9, 2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        kb.verify_drafts(z, t, c, *out, P, ws, draft=draft, uniform=u, uniform_next=last)
    for seed in range(3):
        u.copy_(torch.rand(9, generator=torch.Generator().manual_seed(seed)))
        last.copy_(torch.rand(2, generator=torch.Generator().manual_seed(seed + 50)))
        c[1] = 6 - seed
        g.replay()
        got = [x.tolist() for x in out]
        want = [torch.zeros(n, **I32) for n in (2, 9, 2)]
        kb.verify_drafts(z, t, c, *want, P, ws, draft=draft, uniform=u, uniform_next=last)
        assert got == [x.tolist() for x in want]
