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
