"""The cases on which the key/value-cache, attention and log-probability
operators are measured: their inputs, a plain torch form of each operator, the
calls a user makes, and the same results in 64 bits.

`own` selects what `run` computes: False, the plain form (elementary torch
operations in fp32, rounded once at the end); True, the framework's kernels.
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
        # A prompt's keys and values go into the cache, four requests of odd lengths in one
        # chunk, and are read back (64 query heads share these 8 heads of 64).
        dict(name="write_prompt_int8", op="write", fmt="int8", dtype="f16", heads=8, dim=64,
             block=64, start="0", new="4097,2050,1023,517"),
        # One decode step of 64 requests: each appends one token to a block that is part full.
        dict(name="append_b64_e4m3", op="write", fmt="e4m3", dtype="bf16", heads=8, dim=128,
             block=32, start="spread:64:8191", new="1"),
        # A long stored prefix is taken out of the cache in 16 bits.
        dict(name="read_long_int8", op="read", fmt="int8", dtype="f16", heads=8, dim=128,
             block=64, start="0", new="65521"),
        # Parts of three short requests, starting inside a block.
        dict(name="read_parts_e4m3", op="read", fmt="e4m3", dtype="bf16", heads=8, dim=64,
             block=16, start="5,77,300", new="411,129,7"),
        # One request's next token early in a conversation: latency.
        dict(name="attn_b1_short", op="attn", fmt="int8", dtype="f16", q_heads=64, heads=8,
             dim=64, block=64, start="516", new="1", window=0, sinks=True),
        # One request at the end of a long context: every SM on one sequence.
        dict(name="attn_b1_long", op="attn", fmt="int8", dtype="f16", q_heads=64, heads=8,
             dim=64, block=64, start="131070", new="1", window=0, sinks=True),
        # A serving batch with ragged lengths, 32 query heads on 8 of 128.
        dict(name="attn_b64_ragged", op="attn", fmt="e4m3", dtype="bf16", q_heads=32, heads=8,
             dim=128, block=16, start="spread:64:8191", new="1", window=0, sinks=False),
        # A sliding-window layer of a batch far into its contexts, two guessed tokens each.
        dict(name="attn_b32_window", op="attn", fmt="int8", dtype="bf16", q_heads=64, heads=8,
             dim=64, block=32, start="spread:32:30001", new="2", window=128, sinks=True),
        # Prompt chunks of three requests, each behind a part that is already cached.
        dict(name="attn_prompt", op="attn", fmt="int8", dtype="f16", q_heads=64, heads=8, dim=64,
             block=64, start="1024,3001,4001", new="1024,777,57", window=0, sinks=True),
        # The next token of one request, from the 201088-row lm_head, 20 alternatives.
        dict(name="logprobs_one", op="logprobs", dtype="f16", rows=1, vocab=201088, top=20,
             scale=1.0, masked=0.0),
        # Scoring a prompt: every position of a chunk over the 128256-row lm_head.
        dict(name="logprobs_prompt", op="logprobs", dtype="f16", rows=777, vocab=128256, top=5,
             scale=1.0, masked=0.0),
        # A batch in fp32 at a temperature, most tokens ruled out by a grammar, odd vocabulary.
        dict(name="logprobs_masked_odd", op="logprobs", dtype="f32", rows=37, vocab=50021, top=8,
             scale=1.25, masked=0.9),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "attn", "attn", "logprobs"])
    if op == "logprobs":
        vocab = _log_int(rng, 1000, 201088)
        rows = _log_int(rng, 1, min(4096, 777 * 128256 // vocab))
        dtype = rng.choice(["f16", "bf16", "f32"])
        if dtype == "f32":
            rows = max(1, rows // 2)
        return dict(op=op, dtype=dtype, rows=rows, vocab=vocab, top=rng.choice([1, 5, 8, 20]),
                    scale=rng.choice([1.0, 0.7, 1.25]), masked=rng.choice([0.0, 0.0, 0.9]))
    c = dict(op=op, fmt=rng.choice(["int8", "e4m3"]), dtype=rng.choice(["f16", "bf16"]),
             heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 64, 96, 128, 128]),
             block=rng.choice([16, 32, 64, 128]))
    per_token = c["heads"] * c["dim"]
    if op in ("write", "read"):
        seqs = _log_int(rng, 1, 64)
        most = (8 * 64 * 7687 if op == "write" else 8 * 128 * 65521) // per_token
        if rng.random() < 0.4:
            new = [1] * seqs
        else:
            total = _log_int(rng, seqs, min(most, 40000))
            new = [max(1, int(2 * rng.random() * total / seqs)) for _ in range(seqs)]
            while sum(new) > most:
                new = [max(1, n // 2) for n in new]
        start = [rng.choice([0, rng.randrange(0, 3000)]) for _ in new]
        c.update(start=",".join(map(str, start)), new=",".join(map(str, new)))
        return c
    c.update(q_heads=c["heads"] * rng.choice([1, 4, 5, 8, 16]),
             window=rng.choice([0, 0, 128, 1000]), sinks=rng.random() < 0.5)
    kind = rng.choice(["one", "one", "few", "chunk"])
    if kind == "chunk":
        seqs = rng.randrange(1, 4)
        new = [_log_int(rng, 17, 900) for _ in range(seqs)]
        start = [rng.choice([0, _log_int(rng, 1, 3000)]) for _ in range(seqs)]
    else:
        seqs = _log_int(rng, 1, 64)
        n = 1 if kind == "one" else rng.randrange(2, 9)
        new = [n] * seqs
        most = min(100000, 8 * 64 * 100000 // (per_token * seqs))
        longest = _log_int(rng, 30, max(31, most))
        start = [rng.randrange(0, longest) for _ in range(seqs)]
    c.update(start=",".join(map(str, start)), new=",".join(map(str, new)))
    while work(c)["flops"] > 7e10:                      # the listed prompt's
        new = [max(1, n // 2) for n in new]
        c["new"] = ",".join(map(str, new))
    return c


# ------------------------------------------------------------------ sizes --
def _lengths(case):
    """(start, new) of every sequence.  "spread:n:m" = n starts from 1 to m, unevenly."""
    s = case["start"]
    if s.startswith("spread:"):
        n, m = (int(x) for x in s.split(":")[1:])
        start = [1 + (m - 1) * ((i * 37) % n) // max(1, n - 1) for i in range(n)]
    else:
        start = [int(x) for x in s.split(",")]
    new = [int(x) for x in case["new"].split(",")]
    n = max(len(start), len(new))
    start = start * n if len(start) == 1 else start
    new = new * n if len(new) == 1 else new
    return start, new


def _visible(case):
    """Per sequence: keys that at least one query sees, and query-key pairs."""
    start, new = _lengths(case)
    w = case["window"]
    keys, pairs = 0, 0
    for s, n in zip(start, new):
        lo = max(0, s - w + 1) if w else 0
        keys += s + n - lo
        pairs += sum(min(s + i + 1, w) if w else s + i + 1 for i in range(n))
    return keys, pairs


def work(case):
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        e = 4 if case["dtype"] == "f32" else 2
        return {"bytes": n * e + case["rows"] * (12 + 8 * case["top"]), "flops": 4 * n}
    start, new = _lengths(case)
    H, D, T = case["heads"], case["dim"], sum(new)
    if case["op"] == "attn":
        keys, pairs = _visible(case)
        return {"bytes": 2 * keys * H * D + 4 * T * case["q_heads"] * D,
                "flops": 4 * D * case["q_heads"] * pairs}
    if case["op"] == "read":
        return {"bytes": 2 * T * H * D * 3, "flops": 2 * T * H * D}
    # a write reads 16 bits a value and writes 8; the blocks it touched are then read back
    back = sum(n + s % case["block"] for s, n in zip(start, new))
    return {"bytes": 2 * H * D * (3 * T + 3 * back), "flops": 4 * T * H * D}


# ----------------------------------------------------------------- inputs --
def _round_codes(y, fmt):
    y = y.clamp(-QMAX[fmt], QMAX[fmt])
    return (y.round() if fmt == "int8" else y).to(CODES[fmt])


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    if case["op"] == "logprobs":
        R, V = case["rows"], case["vocab"]
        z = (3.0 * normal(R, V)).to(DTYPES[case["dtype"]])
        tgt = torch.randint(0, V, (R,), device=dev, generator=g, dtype=torch.int32)
        if case["masked"]:
            z[torch.rand(R, V, device=dev, generator=g) < case["masked"]] = -math.inf
        st = dict(case=case, logits=z, targets=tgt)
        if own:
            import kernels_b200 as kb
            P = kb.logprob_params(R, V, case["top"], z.dtype, scale=case["scale"])
            st.update(P=P, ws=kb.LogprobWorkspace(P),
                      out=(torch.empty(R, device=dev), torch.empty(R, device=dev),
                           torch.empty(R, case["top"], device=dev),
                           torch.empty(R, case["top"], device=dev, dtype=torch.int32)))
        return st

    start, new = _lengths(case)
    H, D, bt, fmt, dt = (case["heads"], case["dim"], case["block"], case["fmt"],
                         DTYPES[case["dtype"]])
    B, T = len(new), sum(new)
    # pages of the sequences, in an order that is not theirs
    pages = [-(-(s + n) // bt) for s, n in zip(start, new)]
    total = sum(pages) + 3
    order = torch.randperm(total, device=dev, generator=g).to(torch.int32)
    table = torch.zeros(B, max(pages), dtype=torch.int32, device=dev)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    st = dict(case=case, table=table, start=_ints(start, dev),
              cu=_ints([0] + list(np.cumsum(new)), dev), max_new=max(new),
              max_len=max(s + n for s, n in zip(start, new)))
    # what earlier steps left in the cache: every block with its own scale
    for x in ("k", "v"):
        val = normal(total, H, bt, D) * (0.5 + torch.rand(total, H, 1, 1, device=dev, generator=g))
        s = val.abs().amax(dim=(2, 3)) / QMAX[fmt]
        st[x + "_scale"] = s
        st[x] = _round_codes(val / s[:, :, None, None], fmt)
    if case["op"] == "attn":
        st["q"] = (2.0 * normal(T, case["q_heads"], D)).to(dt)
        st["sinks"] = normal(case["q_heads"]) if case["sinks"] else None
        st["scale"] = D ** -0.5
    elif case["op"] == "write":
        st["new_k"], st["new_v"] = normal(T, H, D).to(dt), normal(T, H, D).to(dt)
        # the blocks that the write touches are read back whole
        back = [(s - s % bt, n + s % bt) for s, n in zip(start, new)]
        st.update(back_start=_ints([s for s, _ in back], dev),
                  back_cu=_ints([0] + list(np.cumsum([n for _, n in back])), dev),
                  back_max=max(n for _, n in back), back_total=sum(n for _, n in back))
    if own:
        import kernels_b200 as kb
        st["cache"] = kb.KVCache(st["k"], st["v"], st["k_scale"], st["v_scale"])
        st["range"] = kb.kv_range(table, st["start"], st["cu"], st["max_new"], st["max_len"])
        if case["op"] == "attn":
            st["P"] = kb.attn_params(case["q_heads"], dt, scale=st["scale"],
                                     window=case["window"])
            st["ws"] = kb.AttnWorkspace(st["cache"], st["range"], st["P"])
            st["out"] = torch.empty_like(st["q"])
            st["lse"] = torch.empty(T, case["q_heads"], device=dev)
        else:
            n = T
            if case["op"] == "write":
                n = st["back_total"]
                st["back"] = kb.kv_range(table, st["back_start"], st["back_cu"], st["back_max"],
                                         st["max_len"])
            st["out"] = (torch.empty(n, H, D, dtype=dt, device=dev),
                         torch.empty(n, H, D, dtype=dt, device=dev))
    return st


# ------------------------------------------------------------ plain forms --
def _places(table, start, cu, block, total):
    """Block, slot in it and sequence of each of the `total` tokens of a range."""
    t = torch.arange(total, device=table.device)
    seq = torch.searchsorted(cu[1:].long(), t, right=True)
    pos = start.long()[seq] + t - cu.long()[seq]
    return table.long()[seq, pos // block], pos % block


def _take(codes, *at):
    """codes[at] in fp32 (8-bit floats are indexed as bytes)."""
    return codes.view(torch.uint8)[at].view(codes.dtype).float()


def _plain_read(st, start, cu, total):
    page, slot = _places(st["table"], start, cu, st["case"]["block"], total)
    dt = DTYPES[st["case"]["dtype"]]
    return [(_take(st[x], page, slice(None), slot) * st[x + "_scale"][page][:, :, None]).to(dt)
            for x in ("k", "v")]


def _plain_write(st):
    case = st["case"]
    bt, fmt, q = case["block"], case["fmt"], QMAX[case["fmt"]]
    start, cu, table = st["start"].long(), st["cu"].long(), st["table"].long()
    page, slot = _places(table, start, cu, bt, st["new_k"].shape[0])
    # the block in which each sequence goes on, and what it holds already
    held = start % bt
    first = table.gather(1, (start // bt)[:, None])[:, 0]
    for x in ("k", "v"):
        new, codes, scale = st["new_" + x].float(), st[x], st[x + "_scale"]
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
    return {"k": k, "v": v, "k_scale": st["k_scale"], "v_scale": st["v_scale"]}


def _plain_attn(st):
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
    p = (start[:, None] + i)[:, :, None]
    see = (j[:, None] <= p) & (i[None, :, None] < n[:, None, None])
    if w:
        see &= j[:, None] > p - w
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


def _plain_logprobs(st):
    case, raw = st["case"], st["logits"]
    z = raw.float() * case["scale"]
    V, k = z.shape[1], case["top"]
    m = z.amax(1, keepdim=True).clamp_min(-3e38)
    e = (z - m).exp()
    L = e.sum(1, keepdim=True)
    lse = m + L.log()
    p = e / L
    # a token without probability adds nothing to the entropy
    ent = -torch.where(p > 0, p * (z - lse), 0.0).sum(1)
    lp = z.gather(1, st["targets"].long()[:, None])[:, 0] - lse[:, 0]
    # ties go to the lowest index: one 64-bit key a token, (value, -index)
    bits = (raw.float() + 0.0).view(torch.int32)
    key = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long() * 2 ** 32
    key += V - 1 - torch.arange(V, device=z.device)
    idx = V - 1 - key.topk(k, dim=1).values.remainder(2 ** 32)
    top = z.gather(1, idx) - lse
    idx = torch.where(top == -math.inf, -1, idx).to(torch.int32)
    return {"logprob": lp, "entropy": ent, "top": top, "index": idx}


def run(state):
    st, op = state, state["case"]["op"]
    if not own:
        if op == "write":
            return _plain_write(st)
        if op == "read":
            k, v = _plain_read(st, st["start"], st["cu"], sum(_lengths(st["case"])[1]))
            return {"k": k, "v": v}
        return _plain_attn(st) if op == "attn" else _plain_logprobs(st)
    import kernels_b200 as kb
    out = st["out"]
    if op == "write":
        kb.kv_write(st["cache"], st["new_k"], st["new_v"], st["range"])
        kb.kv_read(st["cache"], out[0], out[1], st["back"])
        return {"k": out[0], "v": out[1], "k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    if op == "read":
        kb.kv_read(st["cache"], out[0], out[1], st["range"])
        return {"k": out[0], "v": out[1]}
    if op == "attn":
        kb.attn_kv8(st["cache"], st["q"], out, st["range"], st["P"], st["ws"],
                    sinks=st["sinks"], lse=st["lse"])
        return {"out": out, "lse": st["lse"]}
    kb.logprobs(st["logits"], st["targets"], *out, st["P"], st["ws"])
    return {"logprob": out[0], "entropy": out[1], "top": out[2], "index": out[3]}


# ------------------------------------------------------- the same in 64 bits --
def _exact_round(y, fmt):
    """The nearest value that a code can hold (ties to even), in fp64."""
    y = y.clamp(-QMAX[fmt], QMAX[fmt])
    if fmt == "int8":
        return torch.round(y)
    # 3 bits after the leading one; the smallest exponent is -6
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -20))).clamp_min(-6.0) - 3.0)
    return torch.round(y / step) * step


def _exact_tokens(codes, scale, table_row, lo, hi, block):
    pos = torch.arange(lo, hi, device=codes.device)
    blk = table_row.long()[torch.div(pos, block, rounding_mode="floor")]
    raw = codes.view(torch.uint8)[blk, :, pos % block].view(codes.dtype)
    return raw.to(torch.float64) * scale[blk].to(torch.float64).unsqueeze(-1)


def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "logprobs":
        z = st["logits"].to(f64) * float(np.float32(case["scale"]))
        lse = torch.logsumexp(z, 1)
        lp = z[torch.arange(z.shape[0], device=z.device), st["targets"].long()] - lse
        logp = z - lse[:, None]
        ent = -(logp.exp() * logp.masked_fill(logp == -math.inf, 0.0)).sum(1)
        vals, idx = torch.sort(z, dim=1, descending=True, stable=True)
        vals, idx = vals[:, :case["top"]], idx[:, :case["top"]]
        idx = idx.masked_fill(vals == -math.inf, -1).to(torch.int32)
        return {"logprob": lp, "entropy": ent, "top": vals - lse[:, None], "index": idx}
    start, new = _lengths(case)
    bt, H, D = case["block"], case["heads"], case["dim"]
    if case["op"] == "read":
        return {x: torch.cat([_exact_tokens(st[x], st[x + "_scale"], st["table"][b], s, s + n, bt)
                              for b, (s, n) in enumerate(zip(start, new))]) for x in ("k", "v")}
    if case["op"] == "write":
        res = {}
        for x in ("k", "v"):
            fresh = st["new_" + x].to(f64)
            scale, rows, at = st[x + "_scale"].to(f64), [], 0
            for b, (s, n) in enumerate(zip(start, new)):
                done = 0
                while done < n:
                    slot = (s + done) % bt
                    take = min(bt - slot, n - done)
                    blk = int(st["table"][b, (s + done) // bt])
                    part = fresh[at + done:at + done + take]
                    sc = (part.abs().amax(dim=(0, 2)) / QMAX[case["fmt"]]).clamp_min(SCALE_FLOOR)
                    sc = sc.to(torch.float32).to(f64)          # scales are held in 32 bits
                    if slot:
                        was = scale[blk]
                        sc = torch.maximum(sc, was)
                        old = st[x][blk, :, :slot].to(f64).transpose(0, 1)
                        old = _exact_round(old * (was / sc)[None, :, None], case["fmt"])
                        rows.append(old * sc[None, :, None])
                    rows.append(_exact_round(part / sc[None, :, None], case["fmt"])
                                * sc[None, :, None])
                    scale[blk] = sc
                    done += take
                at += n
            res[x], res[x + "_scale"] = torch.cat(rows), scale
        return res
    G, w, outs, lses = case["q_heads"] // H, case["window"], [], []
    at = 0
    for b, (s, n) in enumerate(zip(start, new)):
        lo = max(0, s - w + 1) if w else 0
        K, V = [_exact_tokens(st[x], st[x + "_scale"], st["table"][b], lo, s + n, bt)
                for x in ("k", "v")]
        i = torch.arange(s, s + n, device=K.device)[:, None]
        jj = torch.arange(lo, s + n, device=K.device)[None, :]
        hide = (jj > i) | (jj <= i - w) if w else jj > i
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
