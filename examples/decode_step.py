"""A prompt and decode steps of one gpt-oss-shaped layer on synthetic weights, all
through the library: int4 products for q/k/v, the output projection and the
lm_head, rotary positions on the way to the 8-bit key/value cache, attention over
it, the MoE block, and the log probabilities from which the next token is taken.

    python examples/decode_step.py [--prompt 200] [--steps 8] [--hidden 2880]
        [--vocab 201088] [--experts 16] [--window 128] [--format int8|e4m3]
        [--drafts 7 [--temperature 0.8]]

Prints the prompt's mean log probability and each step's token, with its log
probability, the distribution's entropy and the alternatives.  With --drafts, a
step takes a tree of so many tokens (looked up: what followed the newest token
before, and the likeliest alternatives) through the layer at once, verifies them, and
writes the accepted ones to their places.  Norms and the embedding are a few PyTorch
operations.
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import kernels_b200 as kb                                    # noqa: E402
from kernels_b200 import synth                               # noqa: E402


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def rms(x):
    x = x.float()
    return (x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5)).half()


class Layer:
    """One sequence's layer: weights, cache, and the plans of its calls."""

    def __init__(self, hidden=2880, vocab=201088, q_heads=64, kv_heads=8, dim=64, experts=16,
                 window=0, fmt="int8", block=64, max_len=4096, seed=0):
        self.hidden, self.vocab, self.q_heads, self.kv_heads, self.dim = (hidden, vocab, q_heads,
                                                                          kv_heads, dim)
        rows = (q_heads + 2 * kv_heads) * dim
        self.qkv = synth.int4_weights(rows, hidden, seed=seed)
        self.o = synth.int4_weights(hidden, q_heads * dim, seed=seed + 1)
        self.head = synth.int4_weights(vocab, hidden, seed=seed + 2)
        self.P_qkv, self.P_o = kb.gemv_params(rows, hidden, 64), kb.gemv_params(hidden, q_heads * dim, 64)
        self.P_head = kb.gemv_params(vocab, hidden, 64)
        g = torch.Generator(device="cuda").manual_seed(seed + 3)
        self.embed = torch.randn(vocab, hidden, device="cuda", generator=g, dtype=torch.float16)
        self.sinks = torch.randn(q_heads, device="cuda", generator=g)
        self.P_moe = kb.moe_params(hidden, hidden, experts, 4)
        self.pool, self.R = synth.moe_pool(self.P_moe, seed=seed)
        self.fmt = kb.moe_format(scale_f16=True, has_bias_out=False, act_f16=True, y_f16=True,
                                 n_experts=experts)
        self.ws_moe = kb.MoEWorkspace(self.P_moe)
        blocks = -(-max_len // block)
        self.cache = kb.KVCache.empty(blocks, kv_heads, dim, block,
                                      torch.int8 if fmt == "int8" else torch.float8_e4m3fn)
        self.table = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32)[None]
        # base 150000, 4096 positions scaled by 32
        self.rope = kb.RopeTable(dim, base=150000.0, scaling="yarn", factor=32.0, orig_len=4096.0,
                                 amplitude=1.0 + 0.1 * math.log(32.0))
        self.P_attn = kb.attn_params(q_heads, torch.float16, scale=dim ** -0.5, window=window)
        self.max_len, self.len = max_len, 0
        self.plans = {}

    def plan(self, n):
        """Workspaces of a call on n tokens, made once."""
        if n not in self.plans:
            r = kb.kv_range(self.table, i32([0]), i32([0, n]), n, self.max_len)
            P = kb.logprob_params(n, self.vocab, 5, torch.float16)
            self.plans[n] = (kb.AttnWorkspace(self.cache, r, self.P_attn), P, kb.LogprobWorkspace(P))
        return self.plans[n]

    def product(self, w, P, X):
        """Rows of X through an int4 matrix, 16 at a time."""
        Y = torch.empty(X.shape[0], P.M, dtype=torch.float16, device="cuda")
        for i in range(0, X.shape[0], 16):
            x = X[i:i + 16].contiguous()
            kb.gemm_int4_sb_f16(w["W"], w["SB"], x, Y[i:i + 16], x.shape[0], P)
        return Y

    def qkv_of(self, X):
        """Queries, keys and values, not turned yet."""
        qkv = rms(self.product(self.qkv, self.P_qkv, rms(X)).view(X.shape[0], -1, self.dim))
        return (qkv[:, :self.q_heads], qkv[:, self.q_heads:self.q_heads + self.kv_heads],
                qkv[:, self.q_heads + self.kv_heads:])

    def attend(self, X, start, write=True, tree=None):
        """q/k/v of the tokens at positions start.., turned; their keys and values into
        the cache, attention over everything up to each.  tree: the tokens are a tree
        (mask, positions)."""
        n = X.shape[0]
        q, k, v = self.qkv_of(X)
        r = kb.kv_range(self.table, i32([start]), i32([0, n]), n, self.max_len)
        turned, out = torch.empty_like(q), torch.empty_like(q)
        pos = tree[1] if tree else torch.arange(start, start + n, dtype=torch.int32, device="cuda")
        if write:
            kb.kv_write_rope(self.cache, k, v, r, self.rope, positions=pos, q=q, q_out=turned)
        else:
            kb.rope(q, turned, pos, self.rope)
        if tree:
            kb.attn_tree_kv8(self.cache, turned, out, r, tree[0], self.P_attn, self.plan(n)[0],
                             positions=pos, sinks=self.sinks)
            self.fresh = (k, v, pos, r)      # until it is known which of them stay
        else:
            kb.attn_kv8(self.cache, turned, out, r, self.P_attn, self.plan(n)[0], sinks=self.sinks)
        return out

    def logits(self, tokens, tree=None):
        """The tokens through the layer and the lm_head."""
        X = self.embed[torch.as_tensor(tokens, device="cuda").long()]
        a = self.attend(X, self.len, tree=tree)
        X = X + rms(self.product(self.o, self.P_o, a.reshape(len(tokens), -1)))
        Y = torch.empty_like(X)
        for i, x in enumerate(rms(X)):
            kb.moe_block_ex(self.pool, self.R, x, Y[i], self.P_moe, self.fmt, self.ws_moe)
        X = X + rms(Y)
        return self.product(self.head, self.P_head, rms(X))

    def forward(self, tokens, targets):
        """The tokens through the layer; log probabilities of `targets` after each."""
        n = len(tokens)
        logits = self.logits(tokens)
        self.len += n
        _, P, ws = self.plan(n)
        out = (torch.empty(n, device="cuda"), torch.empty(n, device="cuda"),
               torch.empty(n, 5, device="cuda"), torch.empty(n, 5, dtype=torch.int32, device="cuda"))
        kb.logprobs(logits, i32(targets), *out, P, ws)
        return out

    def step(self, tokens, parents, temperature=0.0, generator=None):
        """A tree of drafted tokens behind the newest one (tokens[0]): the accepted ones,
        the token after them, and the rows of logits.  temperature 0: greedy."""
        n = len(tokens)
        words = -(-n // 32)
        mask, pos = torch.empty(n, words, dtype=torch.int32, device="cuda"), i32([0] * n)
        r = kb.kv_range(self.table, i32([self.len]), i32([0, n]), n, self.max_len)
        par, tok, cu = i32(parents), i32(tokens), i32([0, n])
        kb.draft_tree(par, r, mask, pos, window=self.P_attn.window)
        logits = self.logits(tokens, tree=(mask, pos))
        P = kb.verify_params(1, n, n, self.vocab, torch.float16,
                             scale=1.0 / temperature if temperature else 1.0)
        count, path, last = i32([0]), i32([0] * n), i32([0])
        u = {}
        if temperature:
            u = dict(uniform=torch.rand(n, device="cuda", generator=generator),
                     uniform_next=torch.rand(1, device="cuda", generator=generator))
        kb.verify_drafts(logits, tok, cu, count, path, last, P, kb.VerifyWorkspace(P), parents=par, **u)
        # the accepted tokens' keys and values, to the places that they have without the others
        k, v, pos, r = self.fresh
        kb.kv_write_rope(self.cache, k, v, r, self.rope, positions=pos, rows=path, count=count)
        c = int(count)
        self.len += c
        return path[:c].tolist(), int(last), logits


def generate(layer: Layer, prompt: list[int], steps: int):
    """The prompt in one chunk, then the likeliest token each step."""
    lp, ent, top, idx = layer.forward(prompt, prompt[1:] + [0])
    score = float(lp[:-1].mean()) if len(prompt) > 1 else 0.0
    out = []
    for _ in range(steps):
        tok = int(idx[-1, 0])
        out.append((tok, float(top[-1, 0]), float(ent[-1]), idx[-1].tolist(), top[-1].tolist()))
        lp, ent, top, idx = layer.forward([tok], [tok])
    return score, out


def lookup(history: list[int], alternatives: list[int], drafts: int):
    """A tree behind the newest token: what followed its last earlier occurrence, one after the
    other, and the likeliest alternatives beside the first of these."""
    tokens, parents = [history[-1]], [-1]
    for at in range(len(history) - 2, -1, -1):
        if history[at] == history[-1]:
            for t in history[at + 1:at + 1 + max(1, drafts // 2)]:
                parents.append(len(tokens) - 1)
                tokens.append(t)
            break
    for t in alternatives:
        if len(tokens) > drafts:
            break
        if t not in (x for x, p in zip(tokens, parents) if p == 0):
            parents.append(0)
            tokens.append(t)
    return tokens, parents


def speculate(layer: Layer, prompt: list[int], steps: int, drafts: int, temperature: float = 0.0,
              seed: int = 0):
    """The prompt in one chunk, then trees of drafted tokens: each step's accepted tokens and
    the one drawn after them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    _, _, _, idx = layer.forward(prompt, prompt[1:] + [0])
    history, alternatives = prompt + [int(idx[-1, 0])], idx[-1].tolist()
    out = []
    for _ in range(steps):
        tokens, parents = lookup(history, alternatives, drafts)
        rows, last, logits = layer.step(tokens, parents, temperature, g)
        out.append(([tokens[r] for r in rows], last))
        history += [tokens[r] for r in rows[1:]] + [last]
        alternatives = logits[rows[-1]].topk(5).indices.tolist()
    return out


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--prompt", type=int, default=200)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--hidden", type=int, default=2880)
    ap.add_argument("--vocab", type=int, default=201088)
    ap.add_argument("--experts", type=int, default=16)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--format", choices=["int8", "e4m3"], default="int8")
    ap.add_argument("--drafts", type=int, default=0)
    ap.add_argument("--temperature", type=float, default=0.0)
    a = ap.parse_args()
    layer = Layer(a.hidden, a.vocab, experts=a.experts, window=a.window, fmt=a.format,
                  max_len=a.prompt + (a.steps + 1) * (a.drafts + 1) + 64)
    g = torch.Generator().manual_seed(1)
    prompt = torch.randint(0, a.vocab, (a.prompt,), generator=g).tolist()
    if a.drafts:
        for accepted, last in speculate(layer, prompt, a.steps, a.drafts, a.temperature):
            print(f"accepted {accepted}, then {last}")
        return
    score, out = generate(layer, prompt, a.steps)
    print(f"prompt: {a.prompt} tokens, mean log probability {score:.3f}")
    for tok, lp, ent, idx, top in out:
        alt = ", ".join(f"{i} {t:.2f}" for i, t in zip(idx[1:], top[1:]))
        print(f"token {tok}: log probability {lp:.3f}, entropy {ent:.3f}; next best {alt}")


if __name__ == "__main__":
    main()
