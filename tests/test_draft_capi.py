"""CPU: the entry points of a decode step with drafted tokens refuse bad arguments with
a status before they touch a GPU."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import kernels_b200 as kb
from kernels_b200._lib import AttnParams, RopeDesc, RopeParams, VerifyParams, call
from test_kv_capi import cache, heads, refused, rng


def rope(**kw):
    d = dict(turns=4096, dims=64, layout=0, amplitude=1.0, inverse=0) | kw
    return RopeDesc(*(d[n] for n, _ in RopeDesc._fields_))


def params(**kw):
    d = dict(dims=64, scaling=0, base=1e4, factor=2.0, orig_len=4096.0, low=1.0, high=32.0) | kw
    return RopeParams(*(d[n] for n, _ in RopeParams._fields_))


@pytest.mark.parametrize("match,turns,freqs,p", [
    ("turns must", 0, None, {}), ("turns must", 4104, None, {}), ("freqs must", 4096, 4100, {}),
    ("dims must", 4096, None, dict(dims=24)), ("dims must", 4096, None, dict(dims=0)),
    ("dims must", 4096, None, dict(dims=272)), ("unknown scaling", 4096, None, dict(scaling=4)),
    ("base must", 4096, None, dict(base=0.0)), ("base must", 4096, None, dict(base=float("nan"))),
    ("factor must", 4096, None, dict(scaling=1, factor=0.0)),
    ("orig_len must", 4096, None, dict(scaling=2, low=3.0, high=2.0)),
    ("orig_len must", 4096, None, dict(scaling=3, orig_len=0.0)),
    ("base must not be 1", 4096, None, dict(scaling=2, base=1.0)),
])
def test_rope_tables_refuse(lib, match, turns, freqs, p):
    refused(match, "graft_rope_init", turns, freqs, params(**p), 0)


@pytest.mark.parametrize("match,x,y,n,dim,pos,r", [
    ("16-byte aligned", dict(data=4098), {}, 2, 64, 4096, {}),
    ("element type", dict(dtype=5), {}, 2, 64, 4096, {}),
    ("same type", {}, dict(dtype=1, data=8192), 2, 64, 4096, {}),
    ("same type", {}, dict(tokens=9, data=8192), 2, 64, 4096, {}),
    ("strides", {}, dict(token_stride=132, data=8192), 2, 64, 4096, {}),
    ("must not share memory", {}, dict(token_stride=0, data=8192), 2, 64, 4096, {}),
    ("must not share memory", {}, dict(head_stride=0, data=8192), 2, 64, 4096, {}),
    ("same rows or share no memory", {}, dict(token_stride=256), 2, 64, 4096, {}),
    ("heads", {}, {}, 40000, 64, 4096, {}), ("head_dim", {}, {}, 2, 72, 4096, {}),
    ("head_dim", {}, {}, 2, 272, 4096, {}), ("dims must", {}, {}, 2, 64, 4096, dict(dims=80)),
    ("dims must", {}, {}, 2, 64, 4096, dict(dims=8)), ("unknown layout", {}, {}, 2, 64, 4096, dict(layout=2)),
    ("turns must", {}, {}, 2, 64, 4096, dict(turns=0)),
    ("amplitude", {}, {}, 2, 64, 4096, dict(amplitude=float("inf"))),
    ("positions", {}, {}, 2, 64, 0, {}), ("positions", {}, {}, 2, 64, 4098, {}),
])
def test_rope_refuses(lib, match, x, y, n, dim, pos, r):
    refused(match, "graft_rope", heads(**x), heads(**y), n, dim, pos, rope(**r), 0)


def test_rope_of_nothing(lib):
    for x in (heads(tokens=0), heads(tokens=0, data=0)):
        call("graft_rope", C.byref(x), C.byref(x), 2, 64, 0, C.byref(rope()), 0)
    call("graft_rope", C.byref(heads()), C.byref(heads()), 0, 64, 0, C.byref(rope()), 0)


@pytest.mark.parametrize("match,c,r,extra", [
    ("null buffer", dict(k=0), {}, {}), ("dims must", {}, dict(dims=128), {}),
    ("turns must", {}, dict(turns=8), {}), ("4-byte aligned", {}, {}, dict(pos=4097)),
    ("4-byte aligned", {}, {}, dict(rows=4097, count=4096)), ("go together", {}, {}, dict(rows=4096)),
    ("go together", {}, {}, dict(count=4096)), ("go together", {}, {}, dict(q=heads())),
    ("go together", {}, {}, dict(qo=heads())),
    ("together with rows", {}, {}, dict(q=heads(), qo=heads(), rows=4096, count=4096)),
    ("same type", {}, {}, dict(q=heads(dtype=1), qo=heads(dtype=1))),
    ("same type", {}, {}, dict(q=heads(tokens=7), qo=heads(tokens=7))),
    ("same rows", {}, {}, dict(q=heads(), qo=heads(token_stride=512))),
])
def test_write_rope_refuses(lib, match, c, r, extra):
    e = dict(pos=None, rows=None, count=None, q=None, qo=None) | extra
    q, qo = (None if e[k] is None else C.byref(e[k]) for k in ("q", "qo"))
    refused(match, "graft_kv_write_rope", cache(**c), heads(), heads(), rng(), rope(**r), e["pos"], e["rows"],
            e["count"], q, qo, 2, 0)


@pytest.mark.parametrize("match,args,r", [
    ("parents, mask", dict(parents=0), {}), ("parents, mask", dict(mask=0), {}),
    ("parents, mask", dict(mask=4098), {}), ("parents, mask", dict(positions=4098), {}),
    ("start and cu_tokens", {}, dict(start=0)), ("do not hold", dict(words=0), {}),
    ("do not hold", dict(stride=0), {}), ("do not hold", {}, dict(max_tokens=40)),
    ("max_tokens", {}, dict(max_tokens=65)), ("window", dict(window=1 << 31), {}),
])
def test_draft_tree_refuses(lib, match, args, r):
    a = dict(parents=4096, window=0, mask=4096, stride=1, words=1, positions=None) | args
    refused(match, "graft_draft_tree", a["parents"], rng(**r), 8, a["window"], a["mask"], a["stride"],
            a["words"], a["positions"], 0)


@pytest.mark.parametrize("match,args,p", [
    ("mask must", dict(mask=0), {}), ("mask must", dict(mask=4098), {}),
    ("does not hold", dict(stride=0), {}), ("positions must", {}, dict(window=5)),
    ("positions must", dict(pos=4098), dict(window=5)), ("q_heads", {}, dict(q_heads=3)),
    ("scale", {}, dict(scale=float("inf"))), ("workspace", dict(n=16), {}),
])
def test_tree_attention_refuses(lib, match, args, p):
    a = dict(mask=4096, stride=1, pos=None, n=1 << 40) | args
    P = AttnParams(*(dict(q_heads=4, window=0, scale=1.0) | p).values())
    refused(match, "graft_attn_tree_kv8", cache(), heads(), heads(), rng(), a["mask"], a["stride"], a["pos"],
            None, None, P, 4096, a["n"], 0)


@pytest.mark.parametrize("match,args,p", [
    ("vocab", {}, dict(vocab=0)), ("vocab", {}, dict(vocab=(1 << 30) + 1)), ("max_tokens", {}, dict(max_tokens=1025)), ("element type", {}, dict(dtype=3)),
    ("row stride", {}, dict(row_stride=99)), ("row stride", {}, dict(draft_stride=99)),
    ("scales", {}, dict(scale=0.0)), ("scales", {}, dict(draft_scale=float("nan"))),
    ("tokens", {}, dict(tokens=1 << 27)), ("n_seqs", {}, dict(n_seqs=1 << 25)),
    ("workspace", dict(n=255), {}), ("workspace", dict(ws=4100), {}), ("must be given", dict(cu=0), {}),
    ("must be given", dict(count=0), {}), ("must be given", dict(next=0), {}), ("must be given", dict(path=0), {}),
    ("must be given", dict(tokens=0), {}), ("element type", dict(logits=0), {}),
    ("element type", dict(logits=4097), {}), ("element type", dict(draft=4097), {}),
    ("go together", dict(uniform=0), {}), ("go together", dict(last=0), {}),
    ("4-byte aligned", dict(parents=4097), {}), ("4-byte aligned", dict(uniform=4097), {}),
])
def test_verify_refuses(lib, match, args, p):
    a = dict(logits=4096, draft=4096, tokens=4096, parents=4096, cu=4096, uniform=4096, last=4096, count=4096,
             path=4096, next=4096, ws=4096, n=1 << 40) | args
    d = dict(n_seqs=2, tokens=8, max_tokens=6, vocab=100, dtype=0, row_stride=100, draft_stride=100, scale=1.0,
             draft_scale=1.0) | p
    P = VerifyParams(*(d[n] for n, _ in VerifyParams._fields_))
    refused(match, "graft_verify_drafts", a["logits"], a["draft"], a["tokens"], a["parents"], a["cu"],
            a["uniform"], a["last"], a["count"], a["path"], a["next"], P, a["ws"], a["n"], 0)


def test_sizes_of_the_workspace(lib):
    n = load_ws(1, 6, 201088)
    assert n >= 256 and load_ws(64, 384, 128256) >= n
    assert load_ws(0, 0, 5) == 256


def load_ws(seqs, tokens, vocab):
    return kb.load().graft_verify_workspace(C.byref(kb.verify_params(seqs, tokens, 6, vocab, torch.float16)))


class Table:
    """A rope table that looks as if it were on a GPU."""
    def __init__(self, dev):
        self.dev, self.ref, self.back_ref = dev, None, None


@pytest.fixture
def no_calls(lib, monkeypatch):
    def call(name, *args):
        raise AssertionError(f"{name} was called")
    monkeypatch.setattr(kb, "call", call)


def cpu_case():
    k, s, i = torch.zeros(2, 1, 16, 64, dtype=torch.int8), torch.zeros(2, 1), torch.zeros(1, 1, dtype=torch.int32)
    c = kb.KVCache(k, k.clone(), s, s.clone())
    r = kb.kv_range(i, i[0].clone(), torch.tensor([0, 2], dtype=torch.int32), 2, 2)
    return c, r, torch.zeros(2, 1, 64, dtype=torch.float16)


class Workspace:
    addr, nbytes, dev = 4096, 1 << 30, -1


def test_cpu_tensors_are_refused(no_calls):
    c, r, x = cpu_case()
    i2, m = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="on a GPU"):
        kb.RopeTable(64, device="cpu")
    with pytest.raises(ValueError, match="on a GPU"):
        kb.rope(x, x, i2, Table(-1))
    with pytest.raises(ValueError, match="on a GPU"):
        kb.kv_write_rope(c, x, x, r, Table(-1))
    with pytest.raises(ValueError, match="on a GPU"):
        kb.draft_tree(i2, r, m)
    with pytest.raises(ValueError, match="on a GPU"):
        kb.attn_tree_kv8(c, x, x, r, m, kb.attn_params(1), Workspace())
    P = kb.verify_params(1, 2, 2, 10, torch.float16)
    z, one = torch.zeros(2, 10, dtype=torch.float16), i2[:1].clone()
    with pytest.raises(ValueError, match="on a GPU"):
        kb.verify_drafts(z, i2, i2, one, i2, one, P, Workspace())
    with pytest.raises(ValueError, match="on a GPU"):
        kb.verify_drafts(z, i2, i2, one, i2, one, P, kb.VerifyWorkspace(P, device="cpu"))


def test_shapes_types_and_devices_are_refused(no_calls):
    c, r, x = cpu_case()
    i2, m = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="another device"):
        kb.rope(x, x, i2, Table(0))
    with pytest.raises(ValueError, match="int32"):
        kb.rope(x, x, i2.long(), Table(-1))
    with pytest.raises(ValueError, match="expected a"):
        kb.rope(x, torch.zeros(2, 2, 64).half(), i2, Table(-1))
    with pytest.raises(ValueError, match="tokens, heads, head_dim"):
        kb.rope(x[0], x[0], i2, Table(-1))
    with pytest.raises(ValueError, match="another device"):
        kb.kv_write_rope(c, x, x, r, Table(0))
    with pytest.raises(ValueError, match="go together"):
        kb.kv_write_rope(c, x, x, r, Table(-1), q=x)
    with pytest.raises(ValueError, match="expected a contiguous"):
        kb.kv_write_rope(c, x, x, r, Table(-1), rows=i2, count=i2)
    with pytest.raises(ValueError, match="hold 40 tokens"):
        r40 = kb.kv_range(torch.zeros(1, 9, dtype=torch.int32), i2[:1], i2, 40, 90)
        kb.attn_tree_kv8(c, x, x, r40, m, kb.attn_params(1), Workspace())
    with pytest.raises(ValueError, match="mask must be"):
        kb.attn_tree_kv8(c, x, x, r, m[:1], kb.attn_params(1), Workspace())
    with pytest.raises(ValueError, match="mask must be"):
        kb.draft_tree(i2, r, m[:1])
    with pytest.raises(ValueError, match="unknown layout"):
        kb.RopeTable(64, layout="other")
    with pytest.raises(ValueError, match="unknown scaling"):
        kb.RopeTable(64, scaling="other")
    P = kb.verify_params(1, 2, 2, 10, torch.float16)
    z, one = torch.zeros(2, 10, dtype=torch.float16), i2[:1].clone()
    with pytest.raises(ValueError, match="do not match"):
        kb.verify_drafts(z.float(), i2, i2, one, i2, one, P, Workspace())
    with pytest.raises(ValueError, match="do not match"):
        kb.verify_drafts(z, i2, i2, one, i2, one, P, Workspace(), draft=z[:, :9])
    with pytest.raises(ValueError, match="contiguous"):
        kb.verify_drafts(z, i2, i2, one, i2, one, P, Workspace(), uniform=torch.zeros(3))
    with pytest.raises(TypeError):
        kb.verify_params(1, 2, 2, 10, torch.int8)
