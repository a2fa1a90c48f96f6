"""A prompt and decode steps of one gpt-oss-shaped layer on synthetic weights, all
through the library: int4 products for q/k/v, the output projection and the
lm_head, the 8-bit key/value cache, attention over it, the MoE block, and the
log probabilities from which the next token is taken.

    python examples/decode_step.py [--prompt 200] [--steps 8] [--hidden 2880]
        [--vocab 201088] [--experts 16] [--window 128] [--format int8|e4m3]

Prints the prompt's mean log probability and each step's token, with its log
probability, the distribution's entropy and the alternatives.  Norms, rotary
positions and the embedding are a few PyTorch operations.
"""
from __future__ import annotations

import argparse
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


def rotary(x, pos):
    """x [tokens, heads, dim] turned by the tokens' positions (halves as pairs)."""
    half = x.shape[-1] // 2
    f = 150000.0 ** (-torch.arange(half, device=x.device) / half)
    a = pos[:, None, None].float() * f
    c, s = a.cos(), a.sin()
    x1, x2 = x[..., :half].float(), x[..., half:].float()
    return torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), -1).half()


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

    def attend(self, X, start, write=True):
        """q/k/v of the tokens at positions start.., their keys and values into the
        cache, attention over everything up to each."""
        n = X.shape[0]
        qkv = self.product(self.qkv, self.P_qkv, rms(X)).view(n, -1, self.dim)
        pos = torch.arange(start, start + n, device="cuda")
        q = rotary(rms(qkv[:, :self.q_heads]), pos)
        k = rotary(rms(qkv[:, self.q_heads:self.q_heads + self.kv_heads]), pos)
        v = rms(qkv[:, self.q_heads + self.kv_heads:])
        r = kb.kv_range(self.table, i32([start]), i32([0, n]), n, self.max_len)
        if write:
            kb.kv_write(self.cache, k, v, r)
        out = torch.empty_like(q)
        kb.attn_kv8(self.cache, q, out, r, self.P_attn, self.plan(n)[0], sinks=self.sinks)
        return out

    def forward(self, tokens, targets):
        """The tokens through the layer; log probabilities of `targets` after each."""
        n = len(tokens)
        X = self.embed[torch.as_tensor(tokens, device="cuda")]
        a = self.attend(X, self.len)
        self.len += n
        X = X + rms(self.product(self.o, self.P_o, a.reshape(n, -1)))
        Y = torch.empty_like(X)
        for i, x in enumerate(rms(X)):
            kb.moe_block_ex(self.pool, self.R, x, Y[i], self.P_moe, self.fmt, self.ws_moe)
        X = X + rms(Y)
        logits = self.product(self.head, self.P_head, rms(X))
        _, P, ws = self.plan(n)
        out = (torch.empty(n, device="cuda"), torch.empty(n, device="cuda"),
               torch.empty(n, 5, device="cuda"), torch.empty(n, 5, dtype=torch.int32, device="cuda"))
        kb.logprobs(logits, i32(targets), *out, P, ws)
        return out


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


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--prompt", type=int, default=200)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--hidden", type=int, default=2880)
    ap.add_argument("--vocab", type=int, default=201088)
    ap.add_argument("--experts", type=int, default=16)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--format", choices=["int8", "e4m3"], default="int8")
    a = ap.parse_args()
    layer = Layer(a.hidden, a.vocab, experts=a.experts, window=a.window, fmt=a.format,
                  max_len=a.prompt + a.steps + 64)
    g = torch.Generator().manual_seed(1)
    prompt = torch.randint(0, a.vocab, (a.prompt,), generator=g).tolist()
    score, out = generate(layer, prompt, a.steps)
    print(f"prompt: {a.prompt} tokens, mean log probability {score:.3f}")
    for tok, lp, ent, idx, top in out:
        alt = ", ".join(f"{i} {t:.2f}" for i, t in zip(idx[1:], top[1:]))
        print(f"token {tok}: log probability {lp:.3f}, entropy {ent:.3f}; next best {alt}")


if __name__ == "__main__":
    main()
