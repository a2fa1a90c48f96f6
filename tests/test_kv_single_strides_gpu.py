"""A single token or head, and a table of one block a sequence, may have any stride there."""
from __future__ import annotations

import pytest
import torch

import kernels_b200 as kb

pytestmark = pytest.mark.gpu


def test_strides_of_a_single_token_and_head(lib):
    i32 = dict(dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    for T, H in ((1, 2), (3, 1), (1, 1)):
        flat = torch.randn(4096, device="cuda", generator=g).half()
        # rows 1001 elements apart, heads of a one-head tensor 7: never followed
        odd = flat.as_strided((T, H, 64), (1001 if T == 1 else 64 * H, 7 if H == 1 else 64, 1))
        x = odd.contiguous()
        table, start = torch.tensor([[1]], **i32), torch.zeros(1, **i32)
        r = kb.kv_range(table, start, torch.tensor([0, T], **i32), T, 16)
        a, b = (kb.KVCache.empty(2, H, 64, 16) for _ in range(2))
        kb.kv_write(a, odd, odd, r)
        kb.kv_write(b, x, x, r)
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and bool((a.k != 0).any())
        outs = [torch.zeros(4096, device="cuda").half().as_strided(odd.shape, odd.stride()) for _ in "kvo"]
        want = [torch.zeros_like(x) for _ in "kvo"]
        P = kb.attn_params(H, scale=0.125)
        ws = kb.AttnWorkspace(a, r, P)
        for q, o in ((odd, outs), (x, want)):
            kb.kv_read(a, o[0], o[1], r)
            kb.attn_kv8(a, q, o[2], r, P, ws)
        for o, w in zip(outs, want):
            assert torch.equal(o, w) and bool((w != 0).any())


def test_a_table_of_one_column(lib):
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.arange(12, **i32).view(2, 6).t()[:, 1:]        # 6 sequences, one block each
    assert table.shape == (6, 1) and table.stride(1) != 1
    x = torch.randn(6, 1, 64, device="cuda").half()
    cu, start = torch.arange(7, **i32), torch.zeros(6, **i32)
    a, b = (kb.KVCache.empty(12, 1, 64, 16) for _ in range(2))
    kb.kv_write(a, x, x, kb.kv_range(table, start, cu, 1, 16))
    kb.kv_write(b, x, x, kb.kv_range(table.contiguous(), start, cu, 1, 16))
    assert torch.equal(a.k, b.k) and bool((a.k[6:] != 0).any())
