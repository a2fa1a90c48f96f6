"""CPU: a step in which no sequence has a new token, with host limits that would allow some, is
nothing to do for every entry point of a step with drafted tokens."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import kernels_b200 as kb
from kernels_b200._lib import AttnParams, call
from test_draft_capi import Workspace, rope
from test_kv_capi import cache, heads, rng


@pytest.mark.parametrize("window", [0, 5])
@pytest.mark.parametrize("stride", [0, 1])
def test_tree_attention_without_rows(lib, window, stride):
    x, P = heads(tokens=0, data=0), AttnParams(4, window, 1.0)
    call("graft_attn_kv8", C.byref(cache()), C.byref(x), C.byref(x), C.byref(rng()), None, None, C.byref(P), 4096,
         1 << 40, 0)
    call("graft_attn_tree_kv8", C.byref(cache()), C.byref(x), C.byref(x), C.byref(rng()), 0, stride, 0, None, None,
         C.byref(P), 4096, 1 << 40, 0)


def test_the_other_calls_without_rows(lib):
    x = heads(tokens=0, data=0)
    call("graft_draft_tree", 0, C.byref(rng()), 0, 5, 0, 0, 1, 0, 0)
    call("graft_kv_write_rope", C.byref(cache()), C.byref(x), C.byref(x), C.byref(rng()), C.byref(rope()), None, None,
         None, C.byref(x), C.byref(x), 4, 0)


def test_tree_attention_without_rows_from_python(lib, monkeypatch):
    """The wrapper takes tensors without rows to the library."""
    made = []
    monkeypatch.setattr(kb, "call", lambda name, *args: made.append(name))
    monkeypatch.setattr(kb, "_raw_stream", lambda stream, dev: 0)
    k, s, i = torch.zeros(2, 1, 16, 64, dtype=torch.int8), torch.zeros(2, 1), torch.zeros(1, 1, dtype=torch.int32)
    c = kb.KVCache(k, k.clone(), s, s.clone())
    r = kb.kv_range(i, i[0].clone(), torch.zeros(2, dtype=torch.int32), 8, 16)
    x, none = torch.zeros(0, 1, 64, dtype=torch.float16), torch.zeros(0, dtype=torch.int32)
    mask = torch.zeros(0, 1, dtype=torch.int32)
    kb.draft_tree(none, r, mask, none, window=5)
    kb.attn_tree_kv8(c, x, x, r, mask, kb.attn_params(1, window=5), Workspace(), positions=none)
    assert made == ["graft_draft_tree", "graft_attn_tree_kv8"]
