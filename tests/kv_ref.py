"""Plain 64-bit (numpy) forms of the key/value cache, attention over it and
log probabilities, for the tests."""
from __future__ import annotations

import numpy as np
import torch

QMAX = {"int8": 127.0, "e4m3": 448.0}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# half a unit in the last place, relative: fp16 has 11 significant bits, bf16 8, fp32 24
ROUND = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def f64(t):
    return t.detach().cpu().float().double().numpy()


def make_table(lens, block, n_blocks, rng):
    """Distinct blocks in random order for sequences of `lens` tokens; the rest
    of the table holds numbers that no call may use."""
    need = [-(-n // block) for n in lens]
    order = rng.permutation(n_blocks)[:sum(need)]
    t = np.full((len(lens), max(need + [1]) + 1), 0x7FFFFFF0, np.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return t


def filled_cache(lens, heads, dim, block, fmt, rng, spare=3):
    """A cache in which the sequences' tokens are stored with random codes and
    scales, and all else is what a reused buffer may hold: NaN codes (e4m3),
    NaN scales.  Returns (codes k, v as stored values, scales, table) on the CPU."""
    n_blocks = sum(-(-n // block) for n in lens) + spare
    table = make_table(lens, block, n_blocks, rng)
    used = np.zeros((n_blocks, block), bool)
    for b, n in enumerate(lens):
        for j in range(-(-n // block)):
            used[table[b, j], :min(block, n - j * block)] = True
    res = {}
    for x in ("k", "v"):
        if fmt == "int8":
            c = torch.from_numpy(rng.integers(-127, 128, (n_blocks, heads, block, dim), np.int8))
        else:
            y = rng.normal(0, 60, (n_blocks, heads, block, dim)).clip(-448, 448)
            c = torch.from_numpy(y.astype(np.float32)).to(torch.float8_e4m3fn)
            stale = torch.from_numpy(~used)[:, None, :, None].expand(c.shape)
            c.view(torch.uint8)[stale] = 0x7F
        s = (rng.uniform(0.2, 2.0, (n_blocks, heads)) / QMAX[fmt]).astype(np.float32)
        if fmt == "e4m3":
            s *= 4
        s[~used.any(1)] = np.nan
        res[x], res[x + "_scale"] = c, torch.from_numpy(s)
    return res, torch.from_numpy(table)


def values(cache, x, table, b, n, block):
    """[n, heads, dim] fp64 of sequence b's first n tokens."""
    out = []
    for j in range(-(-n // block)):
        blk = int(table[b, j])
        c = cache[x][blk].float().double().numpy() * float(1)
        out.append((c * cache[x + "_scale"][blk].double().numpy()[:, None, None])
                   .transpose(1, 0, 2)[:min(block, n - j * block)])
    return np.concatenate(out) if out else np.zeros((0,) + tuple(cache[x].shape[1::2]))


def attention(q, K, V, start, scale, window, sinks):
    """q [n, Hq, D], K, V [L, H, D] fp64 -> out, lse, sum_j p_j |v_j|, and the
    largest sum of |products| of a score."""
    n, Hq, D = q.shape
    L, H = K.shape[:2]
    G = Hq // H
    qg = q.reshape(n, H, G, D)
    S = np.einsum("nhgd,lhd->nhgl", qg, K) * scale
    mag = float((np.einsum("nhgd,lhd->nhgl", abs(qg), abs(K)) * abs(scale)).max()) if n and L else 0.0
    p = start + np.arange(n)[:, None]
    j = np.arange(L)[None, :]
    see = (j <= p) & ((j > p - window) if window else True)
    S = np.where(see[:, None, None, :], S, -np.inf)
    if sinks is not None:
        S = np.concatenate([S, np.broadcast_to(sinks.reshape(1, H, G, 1), (n, H, G, 1))], -1)
        V = np.concatenate([V, np.zeros((1, H, D))])
    m = S.max(-1, keepdims=True, initial=-np.inf)
    m = np.where(np.isfinite(m), m, 0.0)
    e = np.exp(S - m)
    l = e.sum(-1, keepdims=True)
    P = np.divide(e, l, out=np.zeros_like(e), where=l > 0)
    with np.errstate(divide="ignore"):
        lse = (m + np.log(l))[..., 0].reshape(n, Hq)
    o = np.einsum("nhgl,lhd->nhgd", P, V).reshape(n, Hq, D)
    a = np.einsum("nhgl,lhd->nhgd", P, abs(V)).reshape(n, Hq, D)
    return o, lse, a, mag
