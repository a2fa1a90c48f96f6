"""Log probabilities, entropy and top alternatives against the formulas in 64
bits.  Indices are exact.  A log probability is z - lse: z has one rounding, lse
the error of a sum of exp (2^-20 relative, each exp and the sums) and of its
own rounding, so the tolerance is 2^-20 (4 + 2 max|z| + |lse|); the entropy
weighs (z - max) by probabilities that are 2^-20 off: 2^-19 (4 + max|z| + sum p |z - max|)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kernels_b200 as kb
from kv_ref import DTYPES

pytestmark = pytest.mark.gpu


def check(logits, k, scale=1.0, targets=None, seed=0):
    R, V = logits.shape
    rng = np.random.default_rng(seed)
    if targets is None:
        targets = rng.integers(0, V, R)
    t = torch.from_numpy(np.asarray(targets, np.int32)).cuda()
    P = kb.logprob_params(R, V, k, logits.dtype, scale=scale)
    ws = kb.LogprobWorkspace(P)
    nan = float("nan")
    lp, ent = torch.full((R,), nan, device="cuda"), torch.full((R,), nan, device="cuda")
    tl = torch.full((R, k), nan, device="cuda")
    ti = torch.full((R, k), -7, dtype=torch.int32, device="cuda")
    kb.logprobs(logits, t, lp, ent, tl, ti, P, ws)
    raw = logits.cpu().double().numpy()
    z = raw * np.float64(np.float32(scale))
    got = [x.cpu().double().numpy() for x in (lp, ent, tl)]
    order = np.argsort(-raw, axis=1, kind="stable")[:, :k]
    vals = np.take_along_axis(z, order, 1)
    want = np.where(vals == -np.inf, -1, order)
    if want.shape[1] < k:      # fewer tokens than alternatives
        want = np.pad(want, ((0, 0), (0, k - want.shape[1])), constant_values=-1)
        vals = np.pad(vals, ((0, 0), (0, k - vals.shape[1])), constant_values=-np.inf)
    assert np.array_equal(ti.cpu().numpy(), want)
    m = z.max(1, keepdims=True)
    none = m[:, 0] == -np.inf
    m = np.where(np.isfinite(m), m, 0)
    e = np.exp(z - m)
    L = np.where(none, 1, e.sum(1))
    lse = m[:, 0] + np.log(L)
    d = np.where(z > -np.inf, z - m, 0)
    E = (e * d).sum(1) / L
    ent64 = np.where(none, 0, np.log(L) - E)
    zmax = np.where(z > -np.inf, abs(z), 0).max(1)
    tol = 2.0 ** -20 * (4 + 2 * zmax + abs(lse))
    lp64 = z[np.arange(R), targets] - lse

    def near(a, b, tol):
        inf = np.isinf(b)
        assert np.array_equal(a[inf], b[inf])
        assert (abs(a[~inf] - b[~inf]) <= np.broadcast_to(tol, b.shape)[~inf]).all()

    near(got[0], lp64, tol)
    near(got[1], ent64, 2.0 ** -19 * (4 + zmax + (e * abs(d)).sum(1) / L))
    near(got[2], vals - lse[:, None], tol[:, None])
    again = [torch.empty_like(x) for x in (lp, ent, tl, ti)]
    kb.logprobs(logits, t, *again, P, ws)
    assert all(torch.equal(a, b) for a, b in zip(again, (lp, ent, tl, ti)))


def normal(R, V, dtype, seed=0, sd=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (sd * torch.randn(R, V, device="cuda", generator=g)).to(DTYPES[dtype])


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("R,V,k", [(1, 1, 1), (3, 2, 5), (2, 31, 32), (5, 257, 1), (1, 201088, 20),
                                   (7, 50021, 8), (300, 1000, 5), (2, 128256, 0), (33, 4099, 32),
                                   (149, 9001, 3)])
def test_random_rows(lib, R, V, k, dtype):
    check(normal(R, V, dtype), k)


@pytest.mark.parametrize("scale", [0.5, 1.25, 1.0 / 0.7, 30.0])
def test_temperature(lib, scale):
    check(normal(4, 3001, "f32"), 10, scale=scale)
    check(normal(4, 3001, "f16"), 10, scale=scale)


def test_unaligned_rows_and_strides(lib):
    buf = normal(9, 5003, "f16", seed=1)
    for lo in range(9):
        check(buf[:, lo:lo + 4001], 7)
    check(normal(18, 777, "f32")[::2, 1:], 4)
    check(normal(5, 1, "bf16")[:, :1], 1)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_ties_go_to_the_lowest_index(lib, dtype):
    z = torch.zeros(3, 20000, device="cuda", dtype=DTYPES[dtype])
    check(z, 32)
    z[1, 7::13] = 2.0
    z[2] = -0.0
    z[2, ::2] = 0.0
    check(z, 20)
    g = torch.Generator(device="cuda").manual_seed(0)
    check(torch.randint(0, 12, (40, 3011), device="cuda", generator=g).to(DTYPES[dtype]), 32)


@pytest.mark.parametrize("order", ["rising", "falling"])
@pytest.mark.parametrize("V", [1000, 30011, 201088])
def test_sorted_logits(lib, V, order):
    z = torch.linspace(-20, 20, V, device="cuda")[None].repeat(2, 1)
    check(z.flip(1).contiguous() if order == "falling" else z, 20)
    check((z.flip(1) if order == "falling" else z).to(torch.float16).contiguous(), 20)


def test_masked_tokens(lib):
    g = torch.Generator(device="cuda").manual_seed(2)
    for dtype in ("f16", "bf16", "f32"):
        z = normal(40, 5001, dtype, seed=3)
        z[torch.rand(40, 5001, device="cuda", generator=g) < 0.97] = -float("inf")
        z[3] = -float("inf")                  # nothing is possible
        z[4] = -float("inf")
        z[4, 4999] = -3.0                     # one token is
        z[5, 3:] = -float("inf")
        check(z, 20)
    z = normal(2, 4096, "f16")                # masks by the type's lowest value
    z[0, 5:] = torch.finfo(torch.float16).min
    z[1] = torch.finfo(torch.float16).min
    check(z, 8)
    z = normal(2, 4096, "f32")
    z[0, 5:] = torch.finfo(torch.float32).min
    z[1] = torch.finfo(torch.float32).min
    check(z, 8)


def test_large_magnitudes(lib):
    z = normal(4, 10001, "f32", sd=1000.0)
    check(z, 5)
    check(normal(4, 10001, "f32", sd=1e30), 5)


def test_nan_and_plus_infinity(lib):
    z = normal(4, 9000, "f32")
    z[1, 77], z[2, 5000] = float("nan"), float("inf")
    R, V, k = 4, 9000, 4
    P = kb.logprob_params(R, V, k, z.dtype)
    ws = kb.LogprobWorkspace(P)
    t = torch.tensor([-1, 3, 5000, V], dtype=torch.int32, device="cuda")
    lp, ent = torch.zeros(R, device="cuda"), torch.zeros(R, device="cuda")
    tl, ti = torch.zeros(R, k, device="cuda"), torch.zeros(R, k, dtype=torch.int32, device="cuda")
    kb.logprobs(z, t, lp, ent, tl, ti, P, ws)
    assert torch.isnan(lp).all()              # no such token, or no such probability
    assert torch.isnan(ent[1:3]).all() and torch.isfinite(ent[[0, 3]]).all()
    assert torch.isnan(tl[1:3]).all() and torch.isfinite(tl[[0, 3]]).all()
    assert (ti >= 0).all() and (ti < V).all() and int(ti[2, 0]) == 5000
    assert not (ti[1] == 77).any()            # a NaN is not an alternative


def test_outputs_may_be_left_out(lib):
    z = normal(6, 7001, "bf16")
    P = kb.logprob_params(6, 7001, 3, z.dtype)
    ws = kb.LogprobWorkspace(P)
    t = torch.arange(6, dtype=torch.int32, device="cuda")
    full = [torch.empty(6, device="cuda"), torch.empty(6, device="cuda"),
            torch.empty(6, 3, device="cuda"), torch.empty(6, 3, dtype=torch.int32, device="cuda")]
    kb.logprobs(z, t, *full, P, ws)
    a = [torch.empty_like(x) for x in full]
    kb.logprobs(z, None, None, None, a[2], a[3], P, ws)
    P0 = kb.logprob_params(6, 7001, 0, z.dtype)
    kb.logprobs(z, t, a[0], a[1], None, None, P0, ws)
    assert all(torch.equal(x, y) for x, y in zip(a, full))


def test_rows_beyond_32_bit_offsets(lib):
    V, R = 201088, 10700                      # 2.15e9 elements
    buf = torch.full((R, V), -4.0, dtype=torch.float16, device="cuda")
    buf[R - 1, 17], buf[R - 1, V - 1] = 9.0, 8.0
    check(buf[R - 2:], 3)
    P = kb.logprob_params(R, V, 2, buf.dtype)
    ws = kb.LogprobWorkspace(P)
    ti = torch.empty(R, 2, dtype=torch.int32, device="cuda")
    tl = torch.empty(R, 2, device="cuda")
    kb.logprobs(buf, None, None, None, tl, ti, P, ws)
    assert ti[R - 1].tolist() == [17, V - 1] and (ti[:R - 1] == torch.tensor([0, 1], device="cuda")).all()
    del buf
    torch.cuda.empty_cache()


def test_graph_and_other_stream(lib):
    for R, V in ((1, 201088), (200, 3001)):
        z = normal(R, V, "f16")
        P = kb.logprob_params(R, V, 5, z.dtype)
        ws = kb.LogprobWorkspace(P)
        t = torch.zeros(R, dtype=torch.int32, device="cuda")
        want = [torch.empty(R, device="cuda"), torch.empty(R, device="cuda"),
                torch.empty(R, 5, device="cuda"), torch.empty(R, 5, dtype=torch.int32, device="cuda")]
        kb.logprobs(z, t, *want, P, ws)
        got = [torch.zeros_like(x) for x in want]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            kb.logprobs(z, t, *got, P, ws)
        for _ in range(3):
            for x in got:
                x.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("rest", [0.0, -1e4, float(torch.finfo(torch.float16).min)])
@pytest.mark.parametrize("V,k", [(5000, 5), (128256, 32)])
def test_most_tokens_share_one_value(lib, V, k, rest):
    z = torch.full((4, V), rest, dtype=torch.float16, device="cuda")
    z[1, V - 1], z[1, 4097], z[1, 11] = 2.0, 1.0, 3.0      # three above the rest
    z[2, ::7] = -float("inf")                              # the first is no token
    z[3, V // 2:] = 1.0                                    # two shared values
    check(z, k)


def test_large_logits_lie_together(lib):
    # every 786 chunks of 8 hold all large logits in their first 31, so that the
    # threads' maxima say little about the k-th largest
    V = 201088
    z = normal(1, V, "f16", sd=1.0)
    z[:, (torch.arange(V, device="cuda") // 8 % 786 % 128) < 31] += 50.0
    check(z, 32)
    check(z.float()[:, :100001], 32)


@pytest.mark.parametrize("above", [960, 1000, 1024, 1100])
def test_many_above_and_many_equal(lib, above):
    # one token's neighbours above a value that all others share: about as many as the
    # collected keys leave room for
    V = 201088
    z = torch.zeros(1, V, dtype=torch.float16, device="cuda")
    at = torch.arange(V, device="cuda")
    few = at[at // 8 % 786 % 128 < 20][:above]
    z[0, few] = 1.0 + torch.arange(above, device="cuda", dtype=torch.float16) / 1024
    check(z, 32)
    check(-z, 32)
