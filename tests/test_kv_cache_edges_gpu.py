"""Ranges that do not rise are reported by the cache's kernels."""
from __future__ import annotations

import pytest
import torch

import kernels_b200 as kb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cu", [[0, 10, 4, 12], [0, 12, 12, 11], [0, -3, 5, 12], [7, 3, 5, 12],
                                [0, 60, 4, 64], [0, 64, 0, 64], [0, 0, 64, 20]])
@pytest.mark.parametrize("read", [False, True])
def test_token_counts_that_do_not_rise_are_reported(lib, read, cu):
    i32 = dict(dtype=torch.int32, device="cuda")
    dev = kb.KVCache.empty(13, 2, 64, 16)
    x = torch.ones(max(cu), 2, 64, device="cuda", dtype=torch.float16)
    table = torch.arange(12, **i32).view(3, 4)
    r = kb.kv_range(table, torch.zeros(3, **i32), torch.tensor(cu, **i32), max(cu), 64)
    kb.kv_device_errors(clear=True)
    if read:
        kb.kv_read(dev, x, x.clone(), r)
    else:
        kb.kv_write(dev, x, x, r)
    assert kb.kv_device_errors(clear=True) == {"block": False, "bounds": True, "wait": False}
    assert (dev.k[12] == 0).all()


def test_a_fall_among_many_sequences_is_reported(lib):
    i32 = dict(dtype=torch.int32, device="cuda")
    n = 1000
    dev = kb.KVCache.empty(n, 1, 64, 16)
    x = torch.ones(n, 1, 64, device="cuda", dtype=torch.float16)
    table = (torch.arange(8 * n, **i32) % n).view(n, 8)
    start = torch.zeros(n, **i32)
    for at in (1, 255, 256, 257, 600, n):
        cu = torch.arange(n + 1, **i32)
        kb.kv_device_errors(clear=True)
        kb.kv_read(dev, x, x, kb.kv_range(table, start, cu, 128, 128))
        assert not any(kb.kv_device_errors().values())
        cu[at] = at - 1 - min(at, 100)      # (the next sequence's 102 tokens are within the bounds)
        kb.kv_read(dev, x, x, kb.kv_range(table, start, cu, 128, 128))
        assert kb.kv_device_errors(clear=True) == {"block": False, "bounds": True, "wait": False}, at
