"""Plain 64-bit (numpy) forms of rotary positions, trees of drafted tokens and
their verification, for the tests."""
from __future__ import annotations

import math

import numpy as np


def frequencies(dims, base=10000.0, scaling="plain", factor=1.0, orig_len=0.0, low=1.0, high=32.0):
    i = np.arange(dims // 2)
    f = base ** (-2.0 * i / dims)
    if scaling == "linear":
        return f / factor
    if scaling == "yarn":
        def at(t):
            return dims * math.log(orig_len / (2 * math.pi * t)) / (2 * math.log(base))
        lo, hi = max(at(high), 0.0), min(at(low), dims - 1.0)
        r = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        return f * (1 - r) + f / factor * r
    if scaling == "bands":
        s = np.clip((orig_len * f / (2 * math.pi) - low) / (high - low), 0, 1)
        return f * s + f / factor * (1 - s)
    return f


def rotate(x, positions, f, layout, amplitude=1.0, inverse=False):
    """x [tokens, heads, dim] fp64 turned; and of each element the magnitude that
    errors of sine and cosine act on, amplitude (|x| + |y|)."""
    half = len(f)
    a = np.asarray(positions, np.float64)[:, None] * f
    c, s = np.cos(a)[:, None] * amplitude, np.sin(a)[:, None] * amplitude * (-1 if inverse else 1)
    y, mag = x.copy(), np.zeros_like(x)
    p, q = (slice(0, half), slice(half, 2 * half)) if layout == "half" else (
        slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    y[..., p] = x[..., p] * c - x[..., q] * s
    y[..., q] = x[..., q] * c + x[..., p] * s
    mag[..., p] = mag[..., q] = abs(amplitude) * (abs(x[..., p]) + abs(x[..., q]))
    return y, mag


def random_parents(n, rng, wide=3):
    return [-1] + [int(rng.integers(max(0, j - 1 - wide * 2), j)) for j in range(1, n)]


def tree_masks(parents, window=0):
    """bool [n, n] (row sees column) and depths."""
    n = len(parents)
    see, depth = np.zeros((n, n), bool), []
    for i, p in enumerate(parents):
        d, j = 0, i
        while True:
            if not window or d < window:
                see[i, j] = True
            p = parents[j]
            if j == 0 or not 0 <= p < j:
                break
            j, d = p, d + 1
        depth.append(d)
    return see, depth


def pack_bits(see, words):
    n = see.shape[0]
    bits = np.zeros((n, words), np.uint32)
    for i, j in zip(*np.nonzero(see)):
        bits[i, j // 32] |= np.uint32(1) << np.uint32(j % 32)
    return bits.view(np.int32)


def tree_attention(q, K, V, start, scale, see, first, sinks):
    """q [n, Hq, D]; K, V [start + n, H, D]: row i sees keys first[i] .. start - 1 and the new
    tokens of see[i].  out, lse, sum_j p_j |v_j|, and the largest sum of |products| of a score."""
    n, Hq, D = q.shape
    L, H = K.shape[:2]
    G = Hq // H
    qg = q.reshape(n, H, G, D)
    S = np.einsum("nhgd,lhd->nhgl", qg, K) * scale
    mag = float((np.einsum("nhgd,lhd->nhgl", abs(qg), abs(K)) * abs(scale)).max())
    seen = np.zeros((n, L), bool)
    seen[:, :start] = np.arange(start)[None, :] >= np.asarray(first)[:, None]
    seen[:, start:] = see
    S = np.where(seen[:, None, None, :], S, -np.inf)
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


def softmax(z, scale):
    """None for a row that gives no distribution."""
    z = z * scale
    m = z.max()
    if not np.isfinite(m) or np.isnan(z).any():
        return None
    e = np.exp(z - m)
    return e / e.sum()


def verify(logits, tokens, parents, scale, draft=None, draft_scale=1.0, uniform=None, last=None):
    """One sequence, fp64.  (accepted rows, next, the smallest relative distance of an
    acceptance to its border, of the draw to its)."""
    n, V = logits.shape
    i, path, near = 0, [0], np.inf
    kids = [[c for c in range(p + 1, n) if parents[c] == p] for p in range(n)]
    greedy = uniform is None
    while True:
        row = logits[i]
        p = softmax(row, scale)
        best = int(np.argmax(row)) if p is not None else -1
        r = None if p is None else p.copy()
        q = softmax(draft[i], draft_scale) if draft is not None and kids[i] else None
        took = None
        for c in kids[i]:
            x = int(tokens[c])
            if not 0 <= x < V or p is None or (draft is not None and q is None and not greedy):
                continue
            if greedy:
                if x == best:
                    took = c
                    break
                continue
            chance = float(uniform[c]) * (q[x] if draft is not None else 1.0) * r.sum()
            if chance or r[x]:
                near = min(near, abs(chance - r[x]) / max(chance, r[x]))
            if chance < r[x]:
                took = c
                break
            if draft is not None:
                r = np.maximum(r - r.sum() * q, 0.0)
            else:
                r[x] = 0.0
            if not r.sum() > 0:
                r = p.copy()
        if took is None:
            break
        i = took
        path.append(i)
    if greedy:
        return path, best, near
    if p is None:
        return path, -1, near
    c = np.cumsum(r)
    goal = float(last) * c[-1]
    ok = np.nonzero((c > goal) & (r > 0))[0]
    near = min(near, float(np.min(np.abs(c - goal))) / c[-1] * 1e6)   # (fp64 sums: 10^6 times finer)
    return path, int(ok[0]) if len(ok) else int(np.nonzero(r > 0)[0][-1]), near
