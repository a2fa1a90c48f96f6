"""Attention over the 8-bit cache where it can go wrong at the edges: windows
without a limit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kernels_b200 as kb
from kv_ref import ROUND, attention, f64
from test_attn_kv8_gpu import attend, cache_of, one_range, run_case

pytestmark = pytest.mark.gpu

INT_MAX = 2 ** 31 - 1


@pytest.mark.parametrize("window", [INT_MAX, INT_MAX - 40, 1 << 30, 701, 700])
def test_windows_beyond_every_sequence(lib, window):
    """The largest int as "no limit": the same bits as no window, for few and many rows."""
    g = torch.Generator(device="cuda").manual_seed(0)
    for H, D in ((2, 64), (1, 128), (1, 256)):
        K, V = (torch.randn(700, H, D, device="cuda", generator=g) for _ in "kv")
        dev, table = cache_of(K, V)
        for start, n in ((699, 1), (690, 10), (0, 200), (300, 400)):
            q = torch.randn(n, 8 * H, D, device="cuda", generator=g).to(torch.float16)
            want = attend(dev, q, one_range(table, start, n), kb.attn_params(8 * H, scale=D ** -0.5))
            got = attend(dev, q, one_range(table, start, n),
                         kb.attn_params(8 * H, scale=D ** -0.5, window=window))
            assert torch.equal(got, want), (H, D, start, n)
    assert not any(kb.kv_device_errors().values())


def test_windows_beyond_the_sequences_of_a_longer_bound(lib):
    """A window that is within max_len and beyond what the sequences hold."""
    run_case([0, 700, 5], [129, 64, 300], 8, 1, 64, 16, "int8", "f16", 1200, False)
