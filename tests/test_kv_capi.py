"""CPU: the cache, attention and log-probability entry points refuse bad
arguments with a status before they touch a GPU, and leave nothing behind."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import kernels_b200 as kb
from kernels_b200 import _lib
from kernels_b200._lib import Heads, KVCacheDesc, KVRangeDesc, call


def cache(**kw):
    d = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, n_blocks=8, kv_heads=2, block_tokens=16,
             head_dim=64, format=0) | kw
    return KVCacheDesc(*(d[n] for n, _ in KVCacheDesc._fields_))


def rng(**kw):
    d = dict(block_table=4096, start=4096, cu_tokens=4096, n_seqs=2, table_stride=4, max_tokens=4,
             max_len=64) | kw
    return KVRangeDesc(*(d[n] for n, _ in KVRangeDesc._fields_))


def heads(**kw):
    d = dict(data=4096, token_stride=128, head_stride=64, tokens=8, dtype=0) | kw
    return Heads(*(d[n] for n, _ in Heads._fields_))


def refused(match, name, *args):
    with pytest.raises(kb.GraftError, match=match) as e:
        call(name, *(C.byref(a) if isinstance(a, C.Structure) else a for a in args))
    assert e.value.code == _lib.GRAFT_EINVAL


@pytest.mark.parametrize("name", ["graft_kv_write", "graft_kv_read"])
@pytest.mark.parametrize("match,c,h,r", [
    ("null buffer", dict(k=0), {}, {}), ("null buffer", dict(v_scale=0), {}, {}),
    ("16-byte aligned", dict(v=4104), {}, {}), ("4-byte aligned", dict(k_scale=4098), {}, {}),
    ("cache format", dict(format=2), {}, {}), ("block_tokens", dict(block_tokens=48), {}, {}),
    ("head_dim", dict(head_dim=72), {}, {}), ("head_dim", dict(head_dim=272), {}, {}),
    ("head_dim", dict(head_dim=0), {}, {}), ("kv_heads", dict(kv_heads=0), {}, {}),
    ("n_blocks", dict(n_blocks=0), {}, {}), ("element type", {}, dict(dtype=3), {}),
    ("16-byte aligned", {}, dict(data=4098), {}), ("16-byte aligned", {}, dict(data=0), {}),
    ("strides", {}, dict(token_stride=132), {}), ("strides", {}, dict(head_stride=68), {}),
    ("null array", {}, {}, dict(block_table=0)), ("null array", {}, {}, dict(cu_tokens=0)),
    ("max_tokens", {}, {}, dict(max_tokens=65)), ("does not hold", {}, {}, dict(table_stride=3)),
    ("4-byte aligned", {}, {}, dict(start=4097)),
])
def test_cache_calls_refuse(lib, name, match, c, h, r):
    refused(match, name, cache(**c), heads(**h), heads(**h), rng(**r), 0)


def test_cache_calls_refuse_unlike_k_and_v(lib):
    refused("same type", "graft_kv_write", cache(), heads(), heads(dtype=1), rng(), 0)
    refused("same type", "graft_kv_read", cache(), heads(), heads(tokens=7), rng(), 0)


@pytest.mark.parametrize("match,p,q,o,more", [
    ("q_heads", dict(q_heads=3), {}, {}, {}), ("q_heads", dict(q_heads=0), {}, {}, {}),
    ("finite", dict(scale=float("nan")), {}, {}, {}), ("finite", dict(scale=float("inf")), {}, {}, {}),
    ("fp16 or both bf16", {}, dict(dtype=2), dict(dtype=2), {}),
    ("fp16 or both bf16", {}, dict(dtype=1), {}, {}),
    ("same number of tokens", {}, {}, dict(tokens=7), {}),
    ("workspace", {}, {}, {}, dict(ws=0)), ("workspace", {}, {}, {}, dict(ws=4096 + 16)),
    ("workspace", {}, {}, {}, dict(n=0)), ("4-byte aligned", {}, {}, {}, dict(lse=4098)),
    ("window", dict(window=1 << 31), {}, {}, {}),
])
def test_attention_refuses(lib, match, p, q, o, more):
    P = _lib.AttnParams(**(dict(q_heads=4, window=0, scale=1.0) | p))
    m = dict(ws=4096, n=1 << 30, lse=0) | more
    refused(match, "graft_attn_kv8", cache(), heads(**q), heads(**o), rng(), None, m["lse"], P,
            m["ws"], m["n"], 0)


def test_workspaces_and_init_refuse(lib):
    P = _lib.AttnParams(3, 0, 1.0)
    assert lib.graft_attn_kv8_workspace(C.byref(cache()), C.byref(rng()), C.byref(P)) == 0
    assert b"q_heads" in lib.graft_last_error_string()
    refused("workspace", "graft_attn_kv8_init", 0, 256, 0)
    refused("workspace", "graft_attn_kv8_init", 4097, 256, 0)
    refused("workspace", "graft_logprobs_init", 0, 256, 0)
    L = _lib.LogprobParams(1, 100, 33, 0, 100, 1.0)
    assert lib.graft_logprobs_workspace(C.byref(L)) == 0


@pytest.mark.parametrize("match,p,a", [
    ("vocab", dict(vocab=0), {}), ("top_k", dict(top_k=33), {}), ("element type", dict(dtype=3), {}),
    ("row_stride", dict(row_stride=99), {}), ("scale", dict(scale=0.0), {}),
    ("scale", dict(scale=-1.0), {}), ("scale", dict(scale=float("nan")), {}),
    ("logits", {}, dict(logits=0)), ("logits", {}, dict(logits=4097)),
    ("go together", {}, dict(targets=0)), ("go together", {}, dict(logprob=0)),
    ("top_logprob", {}, dict(top_lp=0)), ("workspace", {}, dict(ws=0)),
    ("workspace", {}, dict(n=0)),
])
def test_logprobs_refuse(lib, match, p, a):
    P = _lib.LogprobParams(**(dict(rows=2, vocab=100, top_k=4, dtype=0, row_stride=100, scale=1.0) | p))
    m = dict(logits=4096, targets=4096, logprob=4096, entropy=4096, top_lp=4096, top_idx=4096, ws=4096,
             n=1 << 30) | a
    refused(match, "graft_logprobs", m["logits"], m["targets"], m["logprob"], m["entropy"],
            m["top_lp"], m["top_idx"], P, m["ws"], m["n"], 0)


def test_python_wrappers_refuse(lib):
    k = torch.zeros(2, 1, 16, 64, dtype=torch.int8)
    s = torch.zeros(2, 1)
    with pytest.raises(TypeError):
        kb.KVCache(k.to(torch.uint8), k.to(torch.uint8), s, s)
    with pytest.raises(ValueError):
        kb.KVCache(k, k, s.t(), s)
    with pytest.raises(ValueError):
        kb.KVCache(k.transpose(1, 2), k.transpose(1, 2), s, s)
    c = kb.KVCache(k, k, s, s)
    i = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(TypeError):
        kb.kv_range(i.long(), i[0], torch.zeros(2, dtype=torch.int32), 1, 1)
    with pytest.raises(ValueError):
        kb.kv_range(i, i[0], torch.zeros(3, dtype=torch.int32), 1, 1)
    r = kb.kv_range(i, i[0], torch.zeros(2, dtype=torch.int32), 1, 1)
    x = torch.zeros(1, 1, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        kb.kv_write(c, x[:, :, :32], x[:, :, :32], r, stream=0)
    with pytest.raises(ValueError):
        kb.kv_write(c, torch.zeros(1, 1, 128)[:, :, ::2], torch.zeros(1, 1, 64), r, stream=0)
    with pytest.raises(TypeError):
        kb.kv_write(c, x.double(), x.double(), r, stream=0)
    with pytest.raises(TypeError):
        kb.attn_params(8, torch.float32)
    z = torch.zeros(2, 10, dtype=torch.float16)
    P = kb.logprob_params(2, 10, 1, z.dtype)
    with pytest.raises(ValueError):
        kb.logprobs(z[:1], None, None, None, None, None, P, None, stream=0)
    with pytest.raises(ValueError):
        kb.logprobs(z, torch.zeros(2), None, None, None, None, P, None, stream=0)
