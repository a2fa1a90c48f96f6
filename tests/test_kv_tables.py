"""Block tables that are slices of wider ones."""
from __future__ import annotations

import pytest
import torch

import kernels_b200 as kb


def test_a_slice_narrower_than_max_len_is_refused(lib, monkeypatch):
    """The stride of a wider table does not make up for columns that a slice lacks: what
    lies there is another's, or beyond the buffer."""
    def call(name, *args):
        raise AssertionError(f"{name} was called")
    monkeypatch.setattr(kb, "call", call)
    k = torch.zeros(8, 1, 16, 64, dtype=torch.int8)
    s = torch.zeros(8, 1)
    cache = kb.KVCache(k, k.clone(), s, s.clone())
    wide = torch.zeros(2, 8, dtype=torch.int32)
    start, cu = torch.zeros(2, dtype=torch.int32), torch.arange(3, dtype=torch.int32)
    x = torch.zeros(2, 1, 64, dtype=torch.float16)
    P = kb.attn_params(1)

    class ws:
        addr, nbytes, dev = 4096, 1 << 30, -1
    for cols, most, fits in ((slice(0, 4), 64, True), (slice(0, 4), 65, False),
                             (slice(4, 8), 128, False), (slice(6, 8), 33, False),
                             (slice(0, 8), 128, True)):
        r = kb.kv_range(wide[:, cols], start, cu, 1, most)
        want = "on a GPU" if fits else "does not hold max_len"     # (the CPU is refused last)
        for f in (lambda: kb.kv_write(cache, x, x, r), lambda: kb.kv_read(cache, x, x, r),
                  lambda: kb.attn_kv8(cache, x, x, r, P, ws)):
            with pytest.raises(ValueError, match=want):
                f()
    # one sequence: its row's stride says nothing
    r = kb.kv_range(wide[:1, :3], start[:1], cu[:2], 1, 49)
    with pytest.raises(ValueError, match="does not hold max_len"):
        kb.kv_write(cache, x, x, r)


@pytest.mark.gpu
def test_a_slice_of_a_wider_table_works(lib):
    i32 = dict(dtype=torch.int32, device="cuda")
    wide = torch.full((3, 9), -1, **i32)
    wide[:, 2:6] = torch.randperm(12, device="cuda").view(3, 4)
    x = torch.randn(3 * 60, 2, 64, device="cuda").half()
    cu, start = torch.arange(4, **i32) * 60, torch.zeros(3, **i32)
    a, b = (kb.KVCache.empty(12, 2, 64, 16) for _ in range(2))
    kb.kv_write(a, x, x, kb.kv_range(wide[:, 2:6], start, cu, 60, 64))
    kb.kv_write(b, x, x, kb.kv_range(wide[:, 2:6].contiguous(), start, cu, 60, 64))
    assert torch.equal(a.k, b.k) and torch.equal(a.v_scale, b.v_scale)
    assert not any(kb.kv_device_errors().values())
    with pytest.raises((ValueError, kb.GraftError)):
        kb.kv_write(a, x, x, kb.kv_range(wide[:, 2:5], start, cu, 60, 60))
