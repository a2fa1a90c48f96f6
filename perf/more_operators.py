"""The cases on which the operators of a decode step with drafted tokens are
measured: rotary positions, the cache write that applies them, attention of a
tree of drafted tokens over the cache, and their verification.  Their inputs, a
plain torch form of each operator, the calls a user makes, and the same results
in 64 bits.

`own` selects what `run` computes: False, the plain form (elementary torch
operations in fp32, in 64 bits where angles or cumulative sums need them,
rounded once at the end); True, the framework's kernels.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
QMAX = {"int8": 127.0, "e4m3": 448.0}
SCALE_FLOOR = 2.0 ** -64


def listed():
    return [
        # Queries and keys of 16 requests' next tokens, deep in contexts that a scaled rotation
        # reaches: latency.
        dict(name="rope_step", op="rope", dtype="f16", tokens=16, q_heads=64, heads=8, dim=64,
             rot=64, layout="half", scaling="yarn", base=150000.0, far=131072),
        # A prompt's queries and keys, half of each head turned, neighbours as pairs.
        dict(name="rope_prompt", op="rope", dtype="bf16", tokens=7687, q_heads=32, heads=8, dim=128,
             rot=64, layout="interleaved", scaling="plain", base=10000.0, far=8192),
        # A decode step of 64 requests: one token each, its key turned into the cache, its
        # queries turned beside.
        dict(name="write_step_int8", op="write", fmt="int8", dtype="f16", q_heads=64, heads=8,
             dim=64, block=64, rot=64, layout="half", scaling="yarn", base=150000.0,
             start="spread:64:30001", new="1", branch=0),
        # A prompt of four requests of odd lengths, queries included.
        dict(name="write_prompt_int8", op="write", fmt="int8", dtype="f16", q_heads=64, heads=8,
             dim=64, block=64, rot=64, layout="half", scaling="yarn", base=150000.0,
             start="0", new="4097,2050,1023,517", branch=0),
        # The accepted tokens of 32 drafted trees go to their final places.
        dict(name="write_accepted_e4m3", op="write", fmt="e4m3", dtype="bf16", q_heads=0, heads=8,
             dim=128, block=16, rot=128, layout="interleaved", scaling="linear", base=10000.0,
             start="spread:32:8191", new="24", branch=2),
        # One request, a small tree early in a conversation: latency.
        dict(name="tree_b1_short", op="tree", fmt="int8", dtype="f16", q_heads=64, heads=8, dim=64,
             block=64, start="777", new="7", branch=2, window=0, sinks=True),
        # One request at the end of a long context, 64 drafted tokens.
        dict(name="tree_b1_long", op="tree", fmt="int8", dtype="f16", q_heads=64, heads=8, dim=64,
             block=64, start="131001", new="64", branch=3, window=0, sinks=True),
        # A serving batch with ragged lengths, eight tokens in each tree.
        dict(name="tree_b32_ragged", op="tree", fmt="e4m3", dtype="bf16", q_heads=32, heads=8,
             dim=128, block=16, start="spread:32:8191", new="8", branch=2, window=0, sinks=False),
        # A sliding-window layer of a batch, larger trees of several sizes.
        dict(name="tree_b16_window", op="tree", fmt="int8", dtype="bf16", q_heads=64, heads=8,
             dim=64, block=32, start="spread:16:30001", new="32,17,1,24,32,9,32,31,"
             "5,32,27,32,11,32,3,29", branch=2, window=128, sinks=True),
        # One request: five tokens of a draft model after each other, over a 201088-row lm_head.
        dict(name="verify_one", op="verify", dtype="f16", vocab=201088, new="6", branch=1,
             draft=True, scale=1.0, masked=0.0),
        # 64 requests with five drafted tokens each.
        dict(name="verify_b64", op="verify", dtype="f16", vocab=128256, new="6*64", branch=1,
             draft=True, scale=1.0, masked=0.0),
        # Trees whose tokens were looked up (no draft probabilities), at a temperature, most
        # tokens ruled out by a grammar, odd vocabulary, fp32 logits.
        dict(name="verify_trees_odd", op="verify", dtype="f32", vocab=50021, new="31*12,17,1,8,22",
             branch=3, draft=False, scale=1.25, masked=0.9),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(x):
    return ",".join(map(str, x))


def draw(rng):
    op = rng.choice(["rope", "write", "write", "tree", "tree", "verify", "verify"])
    if op == "verify":
        vocab, branch = _log_int(rng, 1000, 201088), rng.choice([1, 1, 2, 3])
        dtype, draft = rng.choice(["f16", "bf16", "f32"]), rng.random() < 0.6
        most = max(2, 384 * 128256 // vocab // (2 if dtype == "f32" else 1))
        seqs = min(_log_int(rng, 1, 64), most // 2)
        longest = rng.choice([2, 4, 6, 9]) if branch == 1 else _log_int(rng, 3, 64)
        new = [max(1, min(rng.randrange(1, longest + 1) if i else longest, most // seqs))
               for i in range(seqs)]
        return dict(op=op, dtype=dtype, vocab=vocab, new=_text(new), branch=branch, draft=draft,
                    scale=rng.choice([1.0, 0.7, 1.25]), masked=rng.choice([0.0, 0.0, 0.9]))
    c = dict(op=op, dtype=rng.choice(["f16", "bf16"]), heads=rng.choice([1, 2, 4, 8]),
             dim=rng.choice([64, 64, 96, 128, 128]))
    if op != "tree":
        c.update(rot=rng.choice([c["dim"], c["dim"], c["dim"] // 2, 16, 32]),
                 layout=rng.choice(["half", "interleaved"]),
                 scaling=rng.choice(["plain", "linear", "yarn", "bands"]),
                 base=rng.choice([10000.0, 150000.0, 500000.0]))
    if op == "rope":
        c.update(dtype=rng.choice(["f16", "bf16", "f32"]),
                 q_heads=c["heads"] * rng.choice([1, 2, 4, 8]),
                 far=_log_int(rng, 100, 1000000))
        c["tokens"] = _log_int(rng, 1, min(8192, 7687 * 40 * 128 * 2 // (
            (c["q_heads"] + c["heads"]) * c["dim"] * (4 if c["dtype"] == "f32" else 2))))
        return c
    c.update(fmt=rng.choice(["int8", "e4m3"]), block=rng.choice([16, 32, 64, 128]))
    seqs = _log_int(rng, 1, 64)
    if op == "write":
        c["q_heads"] = c["heads"] * rng.choice([0, 1, 4, 8])
        most = 7687 * 80 * 64 // ((c["q_heads"] + 2 * c["heads"]) * c["dim"])
        kind = rng.choice(["one", "prompt", "prompt", "accepted"])
        c["branch"] = rng.choice([1, 2, 3]) if kind == "accepted" else 0
        if kind == "one":
            new = [1] * seqs
        else:
            total = _log_int(rng, 2 * seqs, min(most, 40 * seqs if c["branch"] else 20000))
            new = [max(1, int(2 * rng.random() * total / seqs)) for _ in range(seqs)]
            while sum(new) > most:
                new = [max(1, n // 2) for n in new]
        start = [rng.choice([0, rng.randrange(0, 3000)]) for _ in new]
        c.update(start=_text(start), new=_text(new))
        return c
    c.update(q_heads=c["heads"] * rng.choice([1, 4, 5, 8, 16]), branch=rng.choice([1, 2, 3, 4]),
             window=rng.choice([0, 0, 128, 1000]), sinks=rng.random() < 0.5)
    longest = _log_int(rng, 2, 64)
    new = [rng.randrange(1, longest + 1) if i else longest for i in range(seqs)]
    far = _log_int(rng, 30, max(31, min(131001, 8 * 64 * 131001 // (c["heads"] * c["dim"] * seqs))))
    c.update(start=_text([rng.randrange(0, far) for _ in range(seqs)]), new=_text(new))
    while work(c)["flops"] > 1.3e11:                     # the listed long tree's
        far = max(2, far // 2)
        c["start"] = _text([rng.randrange(0, far) for _ in range(seqs)])
    return c


# ------------------------------------------------------------------ sizes --
def _numbers(text):
    """"6*64,3" = 64 times 6, then 3."""
    got = []
    for part in text.split(","):
        x, _, times = part.partition("*")
        got += [int(x)] * int(times or 1)
    return got


def _lengths(case):
    """(start, new) of every sequence.  "spread:n:m" = n starts from 1 to m, unevenly."""
    s = case["start"]
    if s.startswith("spread:"):
        n, m = (int(x) for x in s.split(":")[1:])
        start = [1 + (m - 1) * ((i * 37) % n) // max(1, n - 1) for i in range(n)]
    else:
        start = [int(x) for x in s.split(",")]
    new = _numbers(case["new"])
    n = max(len(start), len(new))
    start = start * n if len(start) == 1 else start
    new = new * n if len(new) == 1 else new
    return start, new


def _parents(n, branch):
    """A tree in which every token has up to `branch` children, level by level."""
    return [(j - 1) // branch if j else -1 for j in range(n)]


def _depths(parents):
    d = []
    for p in parents:
        d.append(d[p] + 1 if p >= 0 else 0)
    return d


def _inner(n, branch):
    """Tokens of such a tree that have children."""
    return -(-(n - 1) // branch)


def _accepted(case):
    """How many tokens of each sequence's tree are written at last: from its root alone
    to a whole branch, in turn."""
    deep = [_depths(_parents(n, case["branch"]))[-1] + 1 for n in _lengths(case)[1]]
    return [1 + (5 * b + 2) % d for b, d in enumerate(deep)]


def work(case):
    if case["op"] == "verify":
        # the rows of tokens with children, of the draft too, and the last accepted token's
        # row where it is a leaf (every second sequence's, say)
        new, e = _numbers(case["new"]), 4 if case["dtype"] == "f32" else 2
        inner = sum(_inner(n, case["branch"]) for n in new)
        n = (inner * (2 if case["draft"] else 1) + len(new) / 2) * case["vocab"]
        return {"bytes": n * e + 20 * sum(new), "flops": 4 * n}
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rope":
        n = case["tokens"] * (case["q_heads"] + case["heads"])
        return {"bytes": 2 * n * case["dim"] * e, "flops": 3 * n * case["rot"]}
    start, new = _lengths(case)
    H, D, T = case["heads"], case["dim"], sum(new)
    if case["op"] == "tree":
        w, G = case["window"], case["q_heads"] // H
        keys = pairs = 0
        for s, n in zip(start, new):
            depth = _depths(_parents(n, case["branch"]))
            keys += n + (min(s, w - 1) if w else s)
            pairs += sum((min(s, w - 1 - d) if w else s) + d + 1 for d in depth)
        return {"bytes": 2 * keys * H * D + 4 * T * H * G * D, "flops": 4 * D * H * G * pairs}
    if case["branch"]:
        new = _accepted(case)
        T = sum(new)
    # keys and values in 16 bits a value to 8, the blocks touched read back, queries in and out
    back = sum(n + s % case["block"] for s, n in zip(start, new))
    return {"bytes": 2 * H * D * (3 * T + 3 * back) + 4 * T * case["q_heads"] * D,
            "flops": (6 * H + 3 * case["q_heads"]) * T * D}


# ----------------------------------------------------------------- inputs --
def _round_codes(y, fmt):
    y = y.clamp(-QMAX[fmt], QMAX[fmt])
    return (y.round() if fmt == "int8" else y).to(CODES[fmt])


def _ints(x, dev="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _sums(x):
    return [0] + [int(n) for n in np.cumsum(x)]


ROPE = {"plain": dict(), "linear": dict(factor=4.0),
        "yarn": dict(factor=32.0, orig_len=4096.0, low=1.0, high=32.0),
        "bands": dict(factor=8.0, orig_len=8192.0, low=1.0, high=4.0)}


def _amplitude(case):
    return 1.0 + 0.1 * math.log(32.0) if case["scaling"] == "yarn" else 1.0


def _frequencies(case):
    """Radians a position of each pair, in 64 bits."""
    n, base, how = case["rot"], case["base"], ROPE[case["scaling"]]
    i = torch.arange(n // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / n)
    if case["scaling"] == "linear":
        return f / how["factor"]
    if case["scaling"] == "yarn":
        # pairs that turn more than `high` times over the first length keep their frequency,
        # those under `low` are slowed down, a ramp between
        def at(turns):
            return n * math.log(how["orig_len"] / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(at(how["high"]), 0.0), min(at(how["low"]), n - 1.0)
        r = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f * (1 - r) + f / how["factor"] * r
    if case["scaling"] == "bands":
        turns = how["orig_len"] * f / (2 * math.pi)
        s = ((turns - how["low"]) / (how["high"] - how["low"])).clamp(0, 1)
        return f * s + f / how["factor"] * (1 - s)
    return f


def _table(case):
    import kernels_b200 as kb
    return kb.RopeTable(case["rot"], base=case["base"], layout=case["layout"],
                        scaling=case["scaling"], amplitude=_amplitude(case),
                        **ROPE[case["scaling"]])


def _prepare_verify(case, normal, g, dev):
    new, V, b = _numbers(case["new"]), case["vocab"], case["branch"]
    B, T, cu = len(new), sum(new), _sums(new)
    st = dict(case=case)
    z = 3.0 * normal(T, V)
    if case["masked"]:
        z[torch.rand(T, V, device=dev, generator=g) < case["masked"]] = -math.inf
    guess = z + 0.7 * normal(T, V)
    seq = torch.repeat_interleave(torch.arange(B), torch.tensor(new))
    i = torch.arange(T) - torch.tensor(cu)[seq]
    parents = torch.where(i > 0, (i - 1) // b, -1).to(dev)
    up = (torch.tensor(cu)[seq].to(dev) + parents.clamp_min(0))     # each token's parent's row
    i = i.to(dev)
    tokens = torch.randint(0, V, (T,), device=dev, generator=g)     # (the roots')
    if case["draft"]:      # drawn from the draft's distribution: the largest of noisy logits
        st["draft"] = guess.to(DTYPES[case["dtype"]])
        for at in range(0, T, 64):      # (a few rows' noise at a time)
            u = torch.rand(up[at:at + 64].numel(), V, device=dev, generator=g)
            noisy = st["draft"][up[at:at + 64]].float() * case["scale"] - u.log_().neg_().log_()
            tokens[at:at + 64] = torch.where(i[at:at + 64] > 0, noisy.argmax(1), tokens[at:at + 64])
            del u, noisy
    else:                  # the likeliest ones of a guess, in turn
        best = guess.topk(b, dim=1).indices
        tokens = torch.where(i > 0, best[up].gather(1, ((i - 1) % b)[:, None])[:, 0], tokens)
    st.update(logits=z.to(DTYPES[case["dtype"]]), tokens=tokens.to(torch.int32), cu=_ints(cu),
              parents=parents.to(torch.int32) if b > 1 else None, levels=_depths(_parents(max(new), b))[-1] + 1, total=T,
              uniform=torch.rand(T, device=dev, generator=g),
              uniform_next=torch.rand(B, device=dev, generator=g))
    if own:
        import kernels_b200 as kb
        P = kb.verify_params(B, T, max(new), V, st["logits"].dtype, scale=case["scale"],
                             draft_scale=case["scale"])
        st.update(P=P, ws=kb.VerifyWorkspace(P), out=tuple(
            torch.empty(n, dtype=torch.int32, device=dev) for n in (B, T, B)))
    return st


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    if case["op"] == "verify":
        return _prepare_verify(case, normal, g, dev)
    H, D, dt, Hq = case["heads"], case["dim"], DTYPES[case["dtype"]], case["q_heads"]
    if case["op"] == "rope":
        T = case["tokens"]
        qkv = normal(T, Hq + 2 * H, D).to(dt)      # (the values' heads stay as they are)
        st = dict(case=case, x=qkv[:, :Hq + H], amplitude=_amplitude(case), positions=torch.randint(
            0, case["far"], (T,), device=dev, generator=g, dtype=torch.int32))
        if own:
            st.update(rope=_table(case), out=torch.empty(T, Hq + H, D, dtype=dt, device=dev))
        return st

    start, new = _lengths(case)
    bt, fmt = case["block"], case["fmt"]
    B, T, cu = len(new), sum(new), _sums(new)
    # pages of the sequences, in an order that is not theirs
    pages = [-(-(s + n) // bt) for s, n in zip(start, new)]
    total = sum(pages) + 3
    order = torch.randperm(total, device=dev, generator=g).to(torch.int32)
    table = torch.zeros(B, max(pages), dtype=torch.int32, device=dev)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    st = dict(case=case, table=table, start=_ints(start), cu=_ints(cu), max_new=max(new),
              max_len=max(s + n for s, n in zip(start, new)), total=T)
    # what earlier steps left in the cache: every block with its own scale
    for x in ("k", "v"):
        val = normal(total, H, bt, D) * (0.5 + torch.rand(total, H, 1, 1, device=dev, generator=g))
        s = val.abs().amax(dim=(2, 3)) / QMAX[fmt]
        st[x + "_scale"] = s
        st[x] = _round_codes(val / s[:, :, None, None], fmt)
    trees = [_parents(n, case["branch"]) for n in new] if case["branch"] else None
    depth = [d for t in trees for d in _depths(t)] if trees else None
    if case["op"] == "tree":
        words = -(-max(new) // 32)
        bits = np.zeros((T, words), np.uint32)
        for c, t in zip(cu, trees):
            for j, p in enumerate(t):
                if p >= 0:
                    bits[c + j] = bits[c + p]
                bits[c + j, j // 32] |= np.uint32(1) << np.uint32(j % 32)
        st.update(mask=torch.from_numpy(bits.view(np.int32)).to(dev),
                  positions=_ints([start[b] + depth[cu[b] + j] for b in range(B)
                                   for j in range(new[b])]),
                  q=(2.0 * normal(T, Hq, D)).to(dt), scale=D ** -0.5,
                  sinks=normal(Hq) if case["sinks"] else None)
    else:
        st["qkv"] = normal(T, Hq + 2 * H, D).to(dt)
        st["new_k"], st["new_v"] = st["qkv"][:, Hq:Hq + H], st["qkv"][:, Hq + H:]
        st["amplitude"], put = _amplitude(case), new
        if trees:       # a path from each root: the rows that stay, and the tokens' places in the tree
            put, rows = _accepted(case), np.full(T, -1, np.int32)
            for b, n in enumerate(put):
                ends = [j for j, d in enumerate(_depths(trees[b])) if d == n - 1]
                j = ends[b % len(ends)]
                for at in range(cu[b] + n - 1, cu[b] - 1, -1):
                    rows[at], j = cu[b] + j, trees[b][j]
            st.update(rows=torch.from_numpy(rows).to(dev), count=_ints(put),
                      positions=_ints([start[b] + depth[cu[b] + j] for b in range(B)
                                       for j in range(new[b])]))
        # the blocks that the write touches are read back whole
        back = [(s - s % bt, n + s % bt) for s, n in zip(start, put)]
        st.update(put_cu=_ints(_sums(put)), put_total=sum(put),
                  back_start=_ints([s for s, _ in back]), back_cu=_ints(_sums([n for _, n in back])),
                  back_max=max(n for _, n in back), back_total=sum(n for _, n in back))
    if own:
        import kernels_b200 as kb
        st["cache"] = kb.KVCache(st["k"], st["v"], st["k_scale"], st["v_scale"])
        st["range"] = kb.kv_range(table, st["start"], st["cu"], st["max_new"], st["max_len"])
        if case["op"] == "tree":
            st["P"] = kb.attn_params(Hq, dt, scale=st["scale"], window=case["window"])
            st["ws"] = kb.AttnWorkspace(st["cache"], st["range"], st["P"])
            st["out"] = torch.empty_like(st["q"])
            st["lse"] = torch.empty(T, Hq, device=dev)
        else:
            st["rope"] = _table(case)
            st["back"] = kb.kv_range(table, st["back_start"], st["back_cu"], st["back_max"],
                                     st["max_len"])
            st["q_out"] = torch.empty(T, Hq, D, dtype=dt, device=dev) if Hq else None
            st["out"] = tuple(torch.empty(st["back_total"], H, D, dtype=dt, device=dev)
                              for _ in range(2))
    return st


# ------------------------------------------------------------ plain forms --
def _plain_rope(x, positions, case, amplitude):
    """x [tokens, heads, dim] turned, in fp32."""
    f, half = _frequencies(case).to(x.device), case["rot"] // 2
    a = positions.double()[:, None] * f
    c, s = (a.cos() * amplitude).float()[:, None], (a.sin() * amplitude).float()[:, None]
    x = x.float()
    t, rest = x[..., :case["rot"]], x[..., case["rot"]:]
    if case["layout"] == "half":
        p, q = t[..., :half], t[..., half:]
        return torch.cat((p * c - q * s, q * c + p * s, rest), -1)
    p, q = t[..., 0::2], t[..., 1::2]
    return torch.cat((torch.stack((p * c - q * s, q * c + p * s), -1).flatten(-2), rest), -1)


def _places(table, start, cu, block, total):
    """Sequence, block and slot in it of each of the `total` tokens of a range."""
    t = torch.arange(total, device=table.device)
    seq = torch.searchsorted(cu[1:].long(), t, right=True)
    pos = start.long()[seq] + t - cu.long()[seq]
    return seq, table.long()[seq, pos // block], pos % block


def _take(codes, *at):
    """codes[at] in fp32 (8-bit floats are indexed as bytes)."""
    return codes.view(torch.uint8)[at].view(codes.dtype).float()


def _plain_read(st, start, cu, total):
    _, page, slot = _places(st["table"], start, cu, st["case"]["block"], total)
    dt = DTYPES[st["case"]["dtype"]]
    return [(_take(st[x], page, slice(None), slot) * st[x + "_scale"][page][:, :, None]).to(dt)
            for x in ("k", "v")]


def _plain_write(st):
    case, q = st["case"], QMAX[st["case"]["fmt"]]
    bt, fmt, dt = case["block"], case["fmt"], DTYPES[st["case"]["dtype"]]
    start, cu, table = st["start"].long(), st["put_cu"].long(), st["table"].long()
    seq, page, slot = _places(table, start, cu, bt, st["put_total"])
    if "rows" in st:
        at = st["cu"].long()[seq] + torch.arange(seq.numel(), device=seq.device) - cu[seq]
        rows = st["rows"].long()[at]
        pos = st["positions"].long()[rows]
    else:
        rows = torch.arange(seq.numel(), device=seq.device)
        pos = start[seq] + rows - cu[seq]
    fresh = {"k": _plain_rope(st["new_k"][rows], pos, case, st["amplitude"]),
             "v": st["new_v"][rows].float()}
    # the block in which each sequence goes on, and what it holds already
    held = start % bt
    first = table.gather(1, (start // bt)[:, None])[:, 0]
    for x, new in fresh.items():
        codes, scale = st[x], st[x + "_scale"]
        amax = torch.zeros_like(scale).index_reduce_(0, page, new.abs().amax(-1), "amax")
        need = (amax / q).clamp_min(SCALE_FLOOR)
        old = scale[first]
        grown = torch.where(held[:, None] > 0, torch.maximum(old, need[first]), need[first])
        scale[page] = need[page]
        scale[first] = grown
        before = codes.view(torch.uint8)[first]
        again = _round_codes(_take(codes, first) * (old / grown)[:, :, None, None], fmt)
        keep = torch.arange(bt, device=table.device)[None, :] < held[:, None]
        codes.view(torch.uint8)[first] = torch.where(keep[:, None, :, None],
                                                     again.view(torch.uint8), before)
        codes.view(torch.uint8)[page, :, slot] = _round_codes(
            new / scale[page][:, :, None], fmt).view(torch.uint8)
    k, v = _plain_read(st, st["back_start"], st["back_cu"], st["back_total"])
    res = {"k": k, "v": v, "k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    if case["q_heads"]:
        res["q"] = _plain_rope(st["qkv"][:, :case["q_heads"]], pos, case, st["amplitude"]).to(dt)
    return res


def _plain_tree(st):
    case, q = st["case"], st["q"]
    bt, w, H, D = case["block"], case["window"], case["heads"], case["dim"]
    G = case["q_heads"] // H
    start, cu, dev = st["start"].long(), st["cu"].long(), q.device
    n, Q = cu[1:] - cu[:-1], st["max_new"]
    # keys lo .. lo + span - 1 of each sequence
    lo = (start - w + 1).clamp_min(0) if w else torch.zeros_like(start)
    span = min(st["max_len"], w + Q - 1) if w else st["max_len"]
    j = lo[:, None] + torch.arange(span, device=dev)
    page = st["table"].long().gather(1, (j // bt).clamp_max(st["table"].shape[1] - 1))
    K, V = [_take(st[x], page, slice(None), j % bt) * st[x + "_scale"][page][..., None]
            for x in ("k", "v")]                                   # [B, span, H, D]
    i = torch.arange(Q, device=dev)
    tok = (cu[:-1, None] + i).clamp_max(q.shape[0] - 1)
    qs = q[tok].float().view(-1, Q, H, G, D).permute(0, 2, 3, 1, 4)  # [B, H, G, Q, D]
    S = torch.matmul(qs.reshape(-1, H, G * Q, D), K.permute(0, 2, 3, 1)) * st["scale"]
    S = S.view(-1, H, G, Q, span)
    # the cached keys by the window, the tree's by the mask
    d = (j - start[:, None])[:, None, :]                           # place in the tree
    words = st["mask"][tok].long()                                 # [B, Q, words]
    at = d.clamp(0, 32 * words.shape[2] - 1).expand(-1, Q, -1)
    bit = (words.gather(2, at // 32) >> (at % 32)) & 1
    see = torch.where(d < 0, True, (bit > 0) & (d < n[:, None, None]))
    if w:
        see &= (d >= 0) | (j[:, None] > st["positions"].long()[tok][:, :, None] - w)
    see &= i[None, :, None] < n[:, None, None]
    S.masked_fill_(~see[:, None, None], -math.inf)
    sink = (st["sinks"] if st["sinks"] is not None else torch.full((H * G,), -math.inf, device=dev))
    sink = sink.view(1, H, G, 1, 1)
    m = torch.maximum(S.amax(-1, keepdim=True), sink).clamp_min(-3e38)
    S = S.sub_(m).exp_()
    L = S.sum(-1, keepdim=True) + (sink - m).exp()
    O = torch.matmul(S.view(-1, H, G * Q, span), V.permute(0, 2, 1, 3)).view(-1, H, G, Q, D)
    O = O / L.clamp_min(1e-38)
    lse = (m + L.log())[..., 0]
    b, i = torch.nonzero(i[None, :] < n[:, None], as_tuple=True)
    O = O.permute(0, 3, 1, 2, 4)[b, i].reshape(-1, H * G, D).to(q.dtype)
    return {"out": O, "lse": lse.permute(0, 3, 1, 2)[b, i].reshape(-1, H * G)}


def _softmax64(z, scale):
    z = z.double() * scale
    e = (z - z.amax(1, keepdim=True)).exp_()
    return e.div_(e.sum(1, keepdim=True))


def _plain_verify(st):
    """All sequences a level of their trees at a time, in 64 bits."""
    case, cu, dev = st["case"], st["cu"].long(), st["logits"].device
    b, B, T = case["branch"], st["cu"].numel() - 1, st["total"]
    n = cu[1:] - cu[:-1]
    now = torch.zeros(B, dtype=torch.long, device=dev)             # the last accepted tokens
    count = torch.ones(B, dtype=torch.long, device=dev)
    path = torch.full((T,), -1, dtype=torch.long, device=dev)
    path[cu[:-1]] = cu[:-1]
    going = torch.ones(B, dtype=torch.bool, device=dev)
    scale = float(np.float32(case["scale"]))
    tokens, u = st["tokens"].long(), st["uniform"].double()
    every = torch.arange(B, device=dev)
    rest = torch.empty(B, case["vocab"], dtype=torch.float64, device=dev)
    for _ in range(st["levels"]):
        row = cu[:-1] + now
        rest = torch.where(going[:, None], _softmax64(st["logits"][row], scale), rest)
        q = _softmax64(st["draft"][row], scale) if case["draft"] else None
        took = torch.zeros_like(going)
        for s in range(b):
            child = b * now + 1 + s
            asks = going & ~took & (child < n)
            at = (cu[:-1] + child).clamp_max(T - 1)
            x, mass = tokens[at], rest.sum(1)
            chance = q[every, x] if q is not None else torch.ones(B, device=dev, dtype=torch.float64)
            yes = asks & (u[at] * chance * mass < rest[every, x])
            no = asks & ~yes
            if q is not None:
                less = (rest - mass[:, None] * q).clamp_min_(0)
            else:
                less = rest.clone()
                less[every, x] = 0
            rest = torch.where(no[:, None], less, rest)
            took |= yes
            path[(cu[:-1] + count)[yes]] = at[yes]
            count += yes
            now = torch.where(yes, child, now)
        going &= took
    c = rest.cumsum(1)
    last = (rest > 0).long().mul_(torch.arange(1, case["vocab"] + 1, device=dev)).amax(1) - 1
    past = (c > st["uniform_next"].double()[:, None] * c[:, -1:]) & (rest > 0)
    nxt = torch.where(past.any(1), past.int().argmax(1), last)
    return {"count": count.int(), "path": path.int(), "next": nxt.int()}


def run(state):
    st, op = state, state["case"]["op"]
    if not own:
        if op == "rope":
            y = _plain_rope(st["x"], st["positions"], st["case"], st["amplitude"])
            return {"x": y.to(st["x"].dtype)}
        return {"write": _plain_write, "tree": _plain_tree, "verify": _plain_verify}[op](st)
    import kernels_b200 as kb
    out = st["out"]
    if op == "rope":
        kb.rope(st["x"], out, st["positions"], st["rope"])
        return {"x": out}
    if op == "write":
        q = st["qkv"][:, :st["case"]["q_heads"]] if st["q_out"] is not None else None
        kb.kv_write_rope(st["cache"], st["new_k"], st["new_v"], st["range"], st["rope"], q=q,
                         q_out=st["q_out"], positions=st.get("positions"), rows=st.get("rows"),
                         count=st.get("count"))
        kb.kv_read(st["cache"], out[0], out[1], st["back"])
        res = {"k": out[0], "v": out[1], "k_scale": st["k_scale"], "v_scale": st["v_scale"]}
        return res if q is None else {**res, "q": st["q_out"]}
    if op == "tree":
        kb.attn_tree_kv8(st["cache"], st["q"], out, st["range"], st["mask"], st["P"], st["ws"],
                         positions=st["positions"], sinks=st["sinks"], lse=st["lse"])
        return {"out": out, "lse": st["lse"]}
    kb.verify_drafts(st["logits"], st["tokens"], st["cu"], *out, st["P"], st["ws"],
                     draft=st.get("draft"), parents=st["parents"], uniform=st["uniform"],
                     uniform_next=st["uniform_next"])
    return {"count": out[0], "path": out[1], "next": out[2]}


# ------------------------------------------------------- the same in 64 bits --
def _exact_round(y, fmt):
    """The nearest value that a code can hold (ties to even), in fp64."""
    y = y.clamp(-QMAX[fmt], QMAX[fmt])
    if fmt == "int8":
        return torch.round(y)
    # 3 bits after the leading one; the smallest exponent is -6
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -20))).clamp_min(-6.0) - 3.0)
    return torch.round(y / step) * step


def _exact_rope(x, positions, case):
    """As complex numbers: each pair times exp(i angle)."""
    x, n = x.to(torch.float64).clone(), case["rot"]
    angle = torch.outer(positions.to(torch.float64), _frequencies(case).to(x.device))
    turn = torch.polar(torch.full_like(angle, _amplitude(case)), angle)[:, None, :]
    if case["layout"] == "half":
        z = torch.complex(x[..., :n // 2].contiguous(), x[..., n // 2:n].contiguous()) * turn
        x[..., :n // 2], x[..., n // 2:n] = z.real, z.imag
    else:
        z = torch.view_as_complex(x[..., :n].unflatten(-1, (-1, 2)).contiguous()) * turn
        x[..., :n] = torch.view_as_real(z).flatten(-2)
    return x


def _exact_tokens(codes, scale, table_row, lo, hi, block):
    pos = torch.arange(lo, hi, device=codes.device)
    blk = table_row.long()[torch.div(pos, block, rounding_mode="floor")]
    raw = codes.view(torch.uint8)[blk, :, pos % block].view(codes.dtype)
    return raw.to(torch.float64) * scale[blk].to(torch.float64).unsqueeze(-1)


def _exact_write(case, st):
    f64, bt, fmt = torch.float64, case["block"], case["fmt"]
    start, new = _lengths(case)
    put = _accepted(case) if case["branch"] else new
    cu, res, fresh = _sums(new), {}, {"k": [], "v": []}
    for b, n in enumerate(put):
        if case["branch"]:
            at = st["rows"][cu[b]:cu[b] + n].long()
            pos = st["positions"][at]
        else:
            at = torch.arange(cu[b], cu[b] + n, device=st["qkv"].device)
            pos = start[b] + at - cu[b]
        fresh["k"].append(_exact_rope(st["new_k"][at], pos, case))
        fresh["v"].append(st["new_v"][at].to(f64))
    for x in ("k", "v"):
        scale, rows = st[x + "_scale"].to(f64), []
        for b, (s, n) in enumerate(zip(start, put)):
            done = 0
            while done < n:
                slot = (s + done) % bt
                take = min(bt - slot, n - done)
                blk = int(st["table"][b, (s + done) // bt])
                part = fresh[x][b][done:done + take]
                sc = (part.abs().amax(dim=(0, 2)) / QMAX[fmt]).clamp_min(SCALE_FLOOR)
                sc = sc.to(torch.float32).to(f64)          # scales are held in 32 bits
                if slot:
                    was = scale[blk]
                    sc = torch.maximum(sc, was)
                    old = st[x][blk, :, :slot].to(f64).transpose(0, 1)
                    rows.append(_exact_round(old * (was / sc)[None, :, None], fmt)
                                * sc[None, :, None])
                rows.append(_exact_round(part / sc[None, :, None], fmt) * sc[None, :, None])
                scale[blk] = sc
                done += take
        res[x], res[x + "_scale"] = torch.cat(rows), scale
    if case["q_heads"]:
        pos = torch.cat([torch.arange(s, s + n) for s, n in zip(start, new)]).to(st["qkv"].device)
        res["q"] = _exact_rope(st["qkv"][:, :case["q_heads"]], pos, case)
    return res


def _exact_tree(case, st):
    f64, start, new = torch.float64, *_lengths(case)
    bt, H, D, w = case["block"], case["heads"], case["dim"], case["window"]
    G, outs, lses, at = case["q_heads"] // H, [], [], 0
    for b, (s, n) in enumerate(zip(start, new)):
        lo = max(0, s - w + 1) if w else 0
        K, V = [_exact_tokens(st[x], st[x + "_scale"], st["table"][b], lo, s + n, bt)
                for x in ("k", "v")]
        # seen: the cached keys that the window leaves, and a token's ancestors
        hide = torch.zeros(n, s + n - lo, dtype=torch.bool)
        parents = _parents(n, case["branch"])
        for i, d in enumerate(_depths(parents)):
            if w:
                hide[i, :max(0, min(s, s + d - w + 1) - lo)] = True
            hide[i, s - lo:] = True
            a = i
            while a >= 0:
                hide[i, s - lo + a] = False
                a = parents[a]
        hide = hide.to(K.device)
        o = torch.empty(n, H * G, D, dtype=f64, device=K.device)
        e = torch.empty(n, H * G, dtype=f64, device=K.device)
        for h in range(H * G):
            x = (st["q"][at:at + n, h].to(f64) @ K[:, h // G].T) * float(st["scale"])
            x = x.masked_fill(hide, -math.inf)
            e[:, h] = torch.logsumexp(x, 1)
            if st["sinks"] is not None:
                e[:, h] = torch.logaddexp(e[:, h], st["sinks"][h].to(f64))
            o[:, h] = torch.exp(x - e[:, h, None]) @ V[:, h // G]
        outs.append(o)
        lses.append(e)
        at += n
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}


def _exact_verify(case, st):
    """One sequence after the other, one row after the other."""
    new, s = _numbers(case["new"]), float(np.float32(case["scale"]))
    cu, path, counts, nexts = _sums(new), np.full(sum(new), -1, np.int32), [], []
    tokens, u = st["tokens"].tolist(), st["uniform"].double().tolist()
    last = st["uniform_next"].double().tolist()

    def row(z):
        return torch.softmax(z.to(torch.float64) * s, 0).cpu().numpy()

    for b, n in enumerate(new):
        parents, i, got = _parents(n, case["branch"]), 0, [0]
        while True:
            p, q, step = row(st["logits"][cu[b] + i]), None, None
            for c in [j for j in range(i + 1, n) if parents[j] == i]:
                x = tokens[cu[b] + c]
                if case["draft"]:
                    q = row(st["draft"][cu[b] + i]) if q is None else q
                else:
                    q = np.zeros_like(p)
                    q[x] = 1.0
                if u[cu[b] + c] * q[x] < p[x]:
                    step = c
                    break
                p = np.maximum(p - q, 0.0) if case["draft"] else np.where(q > 0, 0.0, p)
                p /= p.sum()
            if step is None:
                break
            i = step
            got.append(i)
        path[cu[b]:cu[b] + len(got)] = [cu[b] + j for j in got]
        counts.append(len(got))
        c = np.cumsum(p)
        nexts.append(int(np.nonzero((c > last[b] * c[-1]) & (p > 0))[0][0]))
    return {"count": torch.tensor(counts, dtype=torch.int32), "path": torch.from_numpy(path),
            "next": torch.tensor(nexts, dtype=torch.int32)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        return {"x": _exact_rope(st["x"], st["positions"], case)}
    return {"write": _exact_write, "tree": _exact_tree, "verify": _exact_verify}[case["op"]](case, st)
