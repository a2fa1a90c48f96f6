"""A step with drafted tokens as programs call it beyond the plain cases: queries turned where they lie,
draft rows at other addresses than the target's, captured steps of drawn trees on two streams, and
results compared on every input."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kernels_b200 as kb
from draft_ref import verify
from kv_ref import DTYPES, filled_cache, f64
from test_decode_step_gpu import small
from test_kv_cache_gpu import rng_of, to_dev
from test_verify_gpu import call, expected, make

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device="cuda")

# Both sides are sums in 64 bits: they agree but for random numbers within 2^-40 of a border
# (50021 terms and R down to 2^-10 of them: 2^-53 2^16 2^10 = 2^-27 at the very worst, 2^-40 as a rule,
# and no input here lies nearer than 2^-25).
NEAR = 2.0 ** -25


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dims", [16, 64])
def test_queries_turned_where_they_lie(lib, dims, dtype, layout):
    """q_out is q, a part of one buffer with the keys and values that the call reads."""
    start, new, H, D, bt, Hq = [5, 0, 77, 31], [40, 1, 131, 0], 2, 64, 16, 16
    rng = np.random.default_rng(dims)
    cpu, table = filled_cache([s + m for s, m in zip(start, new)], H, D, bt, "int8", rng)
    here, there = to_dev(cpu), to_dev(cpu)
    T, r, rope = sum(new), rng_of(table, start, new), kb.RopeTable(dims, layout=layout, amplitude=1.25)
    qkv = torch.from_numpy(rng.normal(0, 1, (T, Hq + 2 * H, D)).astype(np.float32)).to(DTYPES[dtype]).cuda()
    own = qkv.clone()
    for positions in (None, torch.from_numpy(rng.integers(0, 9000, T).astype(np.int32)).cuda()):
        q, K, V = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
        out = torch.empty_like(q)
        kb.kv_write_rope(there, K, V, r, rope, positions=positions, q=q, q_out=out)
        mine = own[:, :Hq]
        kb.kv_write_rope(here, own[:, Hq:Hq + H], own[:, Hq + H:], r, rope, positions=positions, q=mine, q_out=mine)
        assert torch.equal(own[:, :Hq], out) and torch.equal(own[:, Hq:], qkv[:, Hq:])
        for x in ("k", "v", "k_scale", "v_scale"):
            assert torch.equal(getattr(here, x).view(torch.uint8), getattr(there, x).view(torch.uint8))
        own.copy_(qkv)
    assert not any(kb.kv_device_errors().values())


def placed(x, at):
    """x's rows with `at` elements before each and an odd distance between them."""
    n, V = x.shape
    wide = torch.zeros(n, (V + at + 1) | 1, dtype=x.dtype, device=x.device)
    wide[:, at:at + V] = x
    return wide[:, at:at + V]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("trees", [True, False])
@pytest.mark.parametrize("at,draft_at", [(0, 1), (3, 0), (2, 7)])
def test_draft_rows_at_other_places(lib, at, draft_at, trees, dtype):
    z, tokens, cu, parents, draft, u, last = make([7, 1, 12, 3], 50021, dtype, at + 10 * draft_at, trees=trees)
    want = expected(z, tokens, cu, parents, 1.0, draft, 1.0, u, last)
    assert min(want[3]) > NEAR
    got = call(placed(z, at), tokens, cu, parents, draft=placed(draft, draft_at), uniform=u, last=last)
    assert got == want[:3]


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("V,dtype", [(999, "f32"), (5003, "f16"), (33000, "bf16")])
def test_every_input_is_compared(lib, V, dtype, drawn):
    """Nothing is drawn again: a random number near a border has to be decided as in 64 bits too."""
    seen = 0
    for seed in range(4):
        z, tokens, cu, parents, draft, u, last = make([31, 1, 17, 64, 2, 9], V, dtype, 100 + seed, drawn=drawn)
        want = expected(z, tokens, cu, parents, 0.8, draft, 0.8, u, last)
        assert min(want[3]) > NEAR
        assert call(z, tokens, cu, parents, 0.8, draft, 0.8, u, last) == want[:3]
        seen += sum(want[0])
    assert seen > 4 * 6


@pytest.mark.parametrize("depth", [5.0, 10.0, 15.0])
def test_siblings_that_leave_little(lib, depth):
    """Two siblings take all but e^-1 to e^-11 of the probability; the third has a thousandth of that."""
    z = torch.full((4, 1000), -depth, device="cuda")
    z[0, 7], z[0, 8] = 3.0, 2.0
    tokens, parents, cu = np.array([0, 7, 8, 500]), np.array([-1, 0, 0, 0]), [0, 4]
    for u, last, n in ((0.0005, 0.3, 2), (0.5, 0.3, 1), (0.0005, 0.99, 2), (0.0012, 0.7, 1)):
        u, last = np.array([0, 0.9999999, 0.9999999, u], np.float32), np.array([last], np.float32)
        want = expected(z, tokens, cu, parents, 1.0, None, 1.0, u, last)
        assert want[3][0] > NEAR and want[0] == [n]
        assert call(z, tokens, cu, parents, uniform=u, last=last) == want[:3]


def test_captured_drawn_trees_on_two_streams(lib):
    """Two captured calls with a cluster a sequence, each with its workspace, replayed side by side on
    inputs that change."""
    sides = []
    for seed, (V, new) in enumerate([(33000, [12, 1, 31, 0, 5]), (70000, [9, 22])]):
        z, tokens, cu, parents, draft, u, last = make(new, V, "f16", 40 + seed)
        P = kb.verify_params(len(new), len(z), max(new), V, z.dtype)
        d = dict(draft=draft, parents=torch.from_numpy(parents).int().cuda(), uniform=torch.from_numpy(u).cuda(),
                 uniform_next=torch.from_numpy(last).cuda())
        sides.append(dict(z=z, t=torch.from_numpy(tokens).int().cuda(), c=torch.tensor(cu, **I32), P=P, d=d, cu=cu,
                          out=[torch.zeros(n, **I32) for n in (len(new), len(z), len(new))],
                          ws=kb.VerifyWorkspace(P), s=torch.cuda.Stream(), g=torch.cuda.CUDAGraph()))
    torch.cuda.synchronize()
    for x in sides:
        with torch.cuda.graph(x["g"], stream=x["s"]):
            kb.verify_drafts(x["z"], x["t"], x["c"], *x["out"], x["P"], x["ws"], **x["d"])
    rng = np.random.default_rng(0)
    for _ in range(3):
        want = []
        for x in sides:
            u, last = rng.random(len(x["z"])).astype(np.float32), rng.random(len(x["cu"]) - 1).astype(np.float32)
            x["d"]["uniform"].copy_(torch.from_numpy(u))
            x["d"]["uniform_next"].copy_(torch.from_numpy(last))
            x["out"][1].fill_(77)
            w = expected(x["z"], x["t"].cpu().numpy().astype(np.int64), x["cu"], x["d"]["parents"].cpu().numpy(), 1.0,
                         x["d"]["draft"], 1.0, u, last)
            assert min(w[3]) > NEAR
            want.append(w[:3])
        torch.cuda.synchronize()
        for _ in range(3):
            for x in sides:
                with torch.cuda.stream(x["s"]):
                    x["g"].replay()
        torch.cuda.synchronize()
        for x, w in zip(sides, want):
            assert tuple(o.tolist() for o in x["out"]) == w


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_every_speculated_step_is_compared(lib, temperature):
    mod, layer = small(lib)
    g = torch.Generator(device="cuda").manual_seed(8)
    prompt = [7, 4999, 12, 12, 3] * 9
    _, _, _, idx = layer.forward(prompt, prompt[1:] + [0])
    history, alternatives = prompt + [int(idx[-1, 0])], idx[-1].tolist()
    for _ in range(12):
        tokens, parents = mod.lookup(history, alternatives, 7)
        again = torch.Generator(device="cuda")
        again.set_state(g.get_state())
        rows, last, logits = layer.step(tokens, parents, temperature, g)
        u = {}
        if temperature:
            u = dict(uniform=torch.rand(len(tokens), device="cuda", generator=again).cpu().numpy(),
                     last=float(torch.rand(1, device="cuda", generator=again)))
        scale = np.float64(np.float32(1.0 / temperature if temperature else 1.0))
        path, nxt, near = verify(f64(logits), tokens, parents, scale, **u)
        assert near > NEAR and rows == path and last == nxt
        history += [tokens[r] for r in rows[1:]] + [last]
        alternatives = logits[rows[-1]].topk(5).indices.tolist()
    assert not any(kb.kv_device_errors().values())
