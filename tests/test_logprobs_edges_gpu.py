"""Log probabilities of logits that lie a step of fp32 apart under a large scale."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kernels_b200 as kb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("low,scale", [(700.0, 1.447e6), (20000.0, 45220.0), (-700.0, 1.447e6),
                                       (1.0, 3.0e8), (3.0e30, 2.0e-23)])
@pytest.mark.parametrize("V", [4096, 9000, 50021])
def test_neighbouring_logits_under_a_large_scale(lib, V, low, scale):
    """Weights are taken against a reference that a thread met first; the neighbour above
    it may lie 2^64 and more above in weight, and must move it.

    lse - z is a sum of 64-bit accuracy but for the exponents: x - ref is exact, its product
    with scale log2(e) is off by 2^-23 of itself, and no exponent that counts passes 2^7, so
    weights are off by 2^-16 and log probabilities by 2^-15 (their own rounding, of numbers
    up to 2^9, is 2^-15 too): 2^-14."""
    up = float(np.nextafter(np.float32(low), np.float32(np.inf)))
    z = torch.full((3, V), low, device="cuda")
    z[0, V // 2:] = up                       # the upper ones after the lower ones
    z[1, :V // 2] = up                       # before them
    z[2, V - 1] = up                         # one alone, the last
    t = torch.tensor([V - 1, 0, V - 1], dtype=torch.int32, device="cuda")
    P = kb.logprob_params(3, V, 4, z.dtype, scale=scale)
    lp, ent, tl = torch.empty(3, device="cuda"), torch.empty(3, device="cuda"), torch.empty(3, 4, device="cuda")
    ti = torch.empty(3, 4, dtype=torch.int32, device="cuda")
    kb.logprobs(z, t, lp, ent, tl, ti, P, kb.LogprobWorkspace(P))
    d = (z.cpu().double().numpy() - up) * np.float64(np.float32(scale))
    lse = np.log(np.exp(d).sum(1))
    p = np.exp(d - lse[:, None])
    assert (abs(lp.cpu().double().numpy() + lse) <= 2.0 ** -14).all()
    assert (abs(tl[:, 0].cpu().double().numpy() + lse) <= 2.0 ** -14).all()
    assert ti[:, 0].tolist() == [V // 2, 0, V - 1]
    want = lse - (p * d).sum(1)
    # the entropy weighs exponents up to 2^9 with those weights
    assert (abs(ent.cpu().double().numpy() - want) <= 2.0 ** -7).all()
