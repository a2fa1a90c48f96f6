"""The cache, attention and log-probability calls take tensors of one GPU, the
current one, and refuse others before anything reaches the library."""
from __future__ import annotations

import pytest
import torch

import kernels_b200 as kb


def cpu_case(dtype=torch.float16):
    k = torch.zeros(2, 1, 16, 64, dtype=torch.int8)
    s = torch.zeros(2, 1)
    i = torch.zeros(1, 1, dtype=torch.int32)
    cache = kb.KVCache(k, k.clone(), s, s.clone())
    r = kb.kv_range(i, i[0].clone(), torch.tensor([0, 1], dtype=torch.int32), 1, 1)
    return cache, r, torch.zeros(1, 1, 64, dtype=dtype)


class Workspace:
    addr, nbytes, dev = 4096, 1 << 30, 0


@pytest.fixture
def no_calls(lib, monkeypatch):
    """Nothing may reach the library."""
    def call(name, *args):
        raise AssertionError(f"{name} was called")
    monkeypatch.setattr(kb, "call", call)


@pytest.mark.parametrize("stream", [None, 0])
def test_cpu_tensors_are_refused(no_calls, stream):
    cache, r, x = cpu_case()
    P = kb.attn_params(1)
    with pytest.raises(ValueError, match="on a GPU"):
        kb.kv_write(cache, x, x, r, stream=stream)
    with pytest.raises(ValueError, match="on a GPU"):
        kb.kv_read(cache, x, x.clone(), r, stream=stream)
    ws = Workspace()
    ws.dev = -1
    with pytest.raises(ValueError, match="on a GPU"):
        kb.attn_kv8(cache, x, x.clone(), r, P, ws, stream=stream)
    with pytest.raises(ValueError, match="on a GPU"):
        kb.AttnWorkspace(cache, r, P)
    z = torch.zeros(2, 10, dtype=torch.float16)
    L = kb.logprob_params(2, 10, 0, z.dtype)
    e = torch.zeros(2)
    with pytest.raises(ValueError, match="on a GPU"):
        kb.logprobs(z, None, None, e, None, None, L, ws, stream=stream)
    with pytest.raises(ValueError, match="on a GPU"):
        kb.LogprobWorkspace(L, device="cpu")


def test_tensors_beside_a_cache_on_a_gpu_are_refused(no_calls):
    """The cache's and the range's device, as it would be on a GPU, set by hand."""
    cache, r, x = cpu_case()
    cache.dev = 0
    with pytest.raises(ValueError, match="cuda:0, not on cpu"):
        kb.kv_write(cache, x, x, r)
    with pytest.raises(ValueError, match="cuda:0, not on cpu"):
        kb.attn_kv8(cache, x, x.clone(), r, kb.attn_params(1), Workspace())
    with pytest.raises(ValueError, match="cuda:0, not on cpu"):
        kb.attn_kv8(cache, x, x.clone(), r, kb.attn_params(1), Workspace(), sinks=torch.zeros(1))
    cache.dev, r.dev = -1, 0
    with pytest.raises(ValueError, match="different devices"):
        kb.kv_read(cache, x, x.clone(), r)


@pytest.mark.gpu
def test_one_cpu_tensor_among_gpu_tensors_is_refused(no_calls):
    cache, r, x = cpu_case()
    g = kb.KVCache(*(getattr(cache, a).cuda() for a in ("k", "v", "k_scale", "v_scale")))
    with pytest.raises(ValueError):
        kb.KVCache(g.k, cache.v, g.k_scale, g.v_scale)
    with pytest.raises(ValueError):
        kb.KVCache(g.k, g.v, g.k_scale, cache.v_scale)
    i = torch.zeros(1, 1, dtype=torch.int32)
    cu = torch.tensor([0, 1], dtype=torch.int32)
    with pytest.raises(ValueError):
        kb.kv_range(i.cuda(), i[0], cu.cuda(), 1, 1)
    with pytest.raises(ValueError):
        kb.kv_range(i.cuda(), i[0].cuda(), cu, 1, 1)
    gr = kb.kv_range(i.cuda(), i[0].cuda(), cu.cuda(), 1, 1)
    gx = x.cuda()
    P, ws, far = kb.attn_params(1), Workspace(), Workspace()
    far.dev = 1
    for bad in (lambda: kb.kv_write(g, x, gx, gr), lambda: kb.kv_write(g, gx, x, gr),
                lambda: kb.kv_write(g, gx, gx, r), lambda: kb.kv_write(cache, gx, gx, gr),
                lambda: kb.attn_kv8(g, x, gx, gr, P, ws), lambda: kb.attn_kv8(g, gx, x, gr, P, ws),
                lambda: kb.attn_kv8(g, gx, gx, gr, P, ws, lse=torch.zeros(1, 1)),
                lambda: kb.attn_kv8(g, gx, gx, gr, P, far)):
        with pytest.raises(ValueError):
            bad()
    z = torch.zeros(2, 10, dtype=torch.float16)
    L = kb.logprob_params(2, 10, 0, z.dtype)
    e = torch.zeros(2)
    for zz, ee, w in ((z, e.cuda(), ws), (z.cuda(), e, ws), (z.cuda(), e.cuda(), far)):
        with pytest.raises(ValueError):
            kb.logprobs(zz, None, None, ee, None, None, L, w)
