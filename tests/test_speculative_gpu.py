"""The decode-step example with trees of drafted tokens: rotary positions, the rotating cache
write, masks, tree attention, verification and the rewrite of accepted tokens together."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kernels_b200 as kb
from draft_ref import verify
from kv_ref import f64
from test_decode_step_gpu import small

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,window", [("int8", 0), ("e4m3", 40)])
def test_a_tree_and_its_paths_agree(lib, fmt, window):
    """A path of the tree attends as the same tokens one after the other do: outputs differ by
    the roundings of both kernels, and of keys that share a block's scale with other tokens."""
    _, layer = small(lib, fmt=fmt, window=window)
    X = layer.embed[torch.arange(100, 160, device="cuda")]
    layer.attend(X, 0)
    parents = [-1, 0, 0, 1, 1, 2, 3, 6]
    Y = layer.embed[torch.tensor([7, 9, 11, 13, 9, 13, 17, 19], device="cuda")]
    r = kb.kv_range(layer.table, torch.tensor([60], dtype=torch.int32, device="cuda"),
                    torch.tensor([0, 8], dtype=torch.int32, device="cuda"), 8, layer.max_len)
    mask, pos = torch.empty(8, 1, dtype=torch.int32, device="cuda"), torch.empty(8, dtype=torch.int32, device="cuda")
    kb.draft_tree(torch.tensor(parents, dtype=torch.int32, device="cuda"), r, mask, pos, window=window)
    assert pos.tolist() == [60, 61, 61, 62, 62, 62, 63, 64]
    tree = layer.attend(Y, 60, tree=(mask, pos))
    vmax = float(tree.abs().max())
    half = 2.0 ** -8 if fmt == "int8" else 2.0 ** -4
    for path in ([0, 1, 3, 6, 7], [0, 2, 5], [0, 1, 4]):
        chain = layer.attend(Y[path], 60)
        # A key's and a value's code is off by half a step (1/254 of the block's largest value, or
        # 2^-4 of itself) in both; q alone is computed again (2^-9 of the largest q).  Scores of magnitude
        # up to dim^1/2 = 8 move by 8 (half + 2^-9) twice; the weights they give by as much.
        assert (chain.float() - tree[path].float()).abs().max() <= vmax * (2 * half + 2 * 8 * (half + 2.0 ** -9))
    assert not any(kb.kv_device_errors().values())


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_speculation(lib, temperature):
    """Every step's path and next token are those of the definition in 64 bits, on the logits
    that the step computed."""
    mod, layer = small(lib)
    g = torch.Generator(device="cuda").manual_seed(3)
    prompt = [7, 4999, 12, 12, 3] * 9
    _, _, _, idx = layer.forward(prompt, prompt[1:] + [0])
    history, alternatives = prompt + [int(idx[-1, 0])], idx[-1].tolist()
    lengths = []
    for i in range(12):
        tokens, parents = mod.lookup(history, alternatives, 7)
        if i % 2:       # a draft that guesses right: what the newest token alone is followed by
            _, guess, _ = layer.step(tokens[:1], [-1])
            layer.len -= 1
            tokens, parents = tokens + [guess, guess], parents + [0, len(tokens)]
        state = g.get_state()
        before = layer.len
        rows, last, logits = layer.step(tokens, parents, temperature, g)
        u = {}
        if temperature:
            again = torch.Generator(device="cuda")
            again.set_state(state)
            u = dict(uniform=torch.rand(len(tokens), device="cuda", generator=again).cpu().numpy(),
                     last=float(torch.rand(1, device="cuda", generator=again)))
        scale = np.float64(np.float32(1.0 / temperature if temperature else 1.0))
        path, nxt, near = verify(f64(logits), tokens, parents, scale, **u)
        if near > 2.0 ** -18:
            assert rows == path and last == nxt
        assert layer.len == before + len(rows)
        history += [tokens[r] for r in rows[1:]] + [last]
        alternatives = logits[rows[-1]].topk(5).indices.tolist()
        lengths.append(len(rows))
    if not temperature:
        assert max(lengths) > 1
    assert not any(kb.kv_device_errors().values())


def test_the_example_runs(lib):
    mod, layer = small(lib)
    out = mod.speculate(layer, [7, 4999, 12, 12, 3] * 9, 5, 7)
    assert len(out) == 5 and all(0 <= t < 5003 for accepted, last in out for t in accepted + [last])
    _, again = small(lib)
    assert mod.speculate(again, [7, 4999, 12, 12, 3] * 9, 5, 7) == out
