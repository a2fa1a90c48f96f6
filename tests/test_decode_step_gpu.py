"""The decode-step example: prompt and decode steps through int4 products, cache,
attention, MoE block and log probabilities together."""
from __future__ import annotations

import math
import sys

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


def small(lib, **kw):
    sys.path.insert(0, str(ROOT / "examples"))
    import decode_step
    args = dict(hidden=256, vocab=5003, q_heads=16, kv_heads=2, dim=64, experts=8, max_len=512, block=32)
    return decode_step, decode_step.Layer(**(args | kw))


@pytest.mark.parametrize("fmt,window", [("int8", 0), ("e4m3", 40)])
def test_a_chunk_and_its_tokens_one_by_one_agree(lib, fmt, window):
    """The many-row and the few-row kernel over the same cache: outputs differ by
    the roundings of both (2^-11 of the output and of the largest value each)."""
    _, layer = small(lib, fmt=fmt, window=window)
    X = layer.embed[torch.arange(100, 190, device="cuda")]
    chunk = layer.attend(X, 0)
    vmax = float(chunk.abs().max())
    for i in (0, 1, 31, 32, 57, 89):
        one = layer.attend(X[i:i + 1], i, write=False)
        # (q alone is computed again: the batched product gives a token the same bits in any batch
        # position up to its summation order, 2^-9 of the largest q, which moves a score of magnitude
        # up to dim^1/2 by 2^-6 at most)
        assert (one[0].float() - chunk[i].float()).abs().max() <= 2.0 ** -6 * vmax
    import kernels_b200 as kb
    assert not any(kb.kv_device_errors().values())


def test_generation(lib):
    mod, layer = small(lib)
    prompt = [7, 4999, 12, 12, 3] * 9
    score, out = mod.generate(layer, prompt, 12)
    assert layer.len == len(prompt) + 12
    assert -2 * math.log(5003) - 40 < score < 0
    for tok, lp, ent, idx, top in out:
        assert tok == idx[0] and 0 <= tok < 5003 and lp == top[0]
        assert all(a >= b for a, b in zip(top, top[1:])) and len(set(idx)) == 5
        assert sum(math.exp(t) for t in top) <= 1 + 1e-5
        assert 0 <= ent <= math.log(5003) + 1e-5
    # the likeliest token's log probability as a target is the same number
    _, again = small(lib)
    score2, out2 = mod.generate(again, prompt, 12)
    assert score2 == score and out2 == out
