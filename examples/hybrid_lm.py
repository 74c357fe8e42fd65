"""A small language model of a selective state space block and a gated linear attention block with
normed, rotated queries and keys: trained on a synthetic task, then served token by token.

    python examples/hybrid_lm.py [--steps 1000]

The task: a sequence of random symbols, a separator, and the same symbols again; the loss counts
the second half. Serving runs prompts of different lengths packed into one row, keeps their states
in slots of a pool, and continues all of them one token at a time.
"""

import argparse
import os
import sys

import torch
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..",
                                "pallas-kernel_amd"))

from tops.ops.gla import chunk_gla, fused_recurrent_gla   # noqa: E402
from tops.ops.rope import qk_norm_rope, rotary_inv_freq   # noqa: E402
from tops.ops.ssm import (causal_conv1d, causal_conv1d_step, selective_scan,   # noqa: E402
                          selective_scan_step)


def positions_of(cu, device):
    return torch.cat([torch.arange(b - a) for a, b in zip(cu, cu[1:])]).to(device)[None]


class SelectiveBlock(nn.Module):
    """Input projection, short convolution, selective scan, output projection."""

    def __init__(self, width, inner, state_size=16, conv_width=4):
        super().__init__()
        self.inner, self.N, self.W = inner, state_size, conv_width
        self.rank = max(1, inner // 16)
        self.norm = nn.RMSNorm(width)
        self.in_proj = nn.Linear(width, 2 * inner, bias=False)
        self.conv = nn.Parameter(torch.randn(inner, conv_width) * conv_width ** -0.5)
        self.conv_bias = nn.Parameter(torch.zeros(inner))
        self.bc_proj = nn.Linear(inner, self.rank + 2 * state_size, bias=False)
        self.dt_proj = nn.Linear(self.rank, inner, bias=False)
        self.A_log = nn.Parameter(torch.log(torch.arange(1.0, state_size + 1)).repeat(inner, 1))
        self.D = nn.Parameter(torch.ones(inner))
        dt = torch.exp(torch.empty(inner).uniform_(-6.9, -2.3))   # steps of 0.001 .. 0.1
        self.dt_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))
        self.out_proj = nn.Linear(inner, width, bias=False)

    def _scan_inputs(self, x):
        dt, B, C = self.bc_proj(x).split([self.rank, self.N, self.N], -1)
        return self.dt_proj(dt), -torch.exp(self.A_log.float()), B, C, self.D

    def forward(self, h, cu=None, keep=False):
        x, z = self.in_proj(self.norm(h)).chunk(2, -1)
        x, window = causal_conv1d(x, self.conv, self.conv_bias, activation="silu",
                                  output_final_state=keep, cu_seqlens=cu)
        y, state = selective_scan(x, *self._scan_inputs(x), z=z, delta_bias=self.dt_bias,
                                  delta_softplus=True, output_final_state=keep, cu_seqlens=cu)
        return h + self.out_proj(y), (window, state)

    def empty_pool(self, slots, like):
        return (like.new_zeros(slots, self.W, self.inner),
                torch.zeros(slots, self.inner, self.N, device=like.device))

    def step(self, h, pool, slots):
        x, z = self.in_proj(self.norm(h)).chunk(2, -1)
        x = causal_conv1d_step(x, pool[0], self.conv, self.conv_bias, activation="silu",
                               state_indices=slots)
        y = selective_scan_step(pool[1], x, *self._scan_inputs(x), z=z, delta_bias=self.dt_bias,
                                delta_softplus=True, state_indices=slots)
        return h + self.out_proj(y)


class AttentionBlock(nn.Module):
    """Gated linear attention of queries and keys that are normed for each head and rotated."""

    def __init__(self, width, heads):
        super().__init__()
        self.heads, self.dim = heads, width // heads
        self.norm = nn.RMSNorm(width)
        self.qkv = nn.Linear(width, 3 * width, bias=False)
        self.gate = nn.Linear(width, width, bias=True)
        self.q_weight = nn.Parameter(torch.ones(self.dim))
        self.k_weight = nn.Parameter(torch.ones(self.dim))
        self.out_proj = nn.Linear(width, width, bias=False)
        self.register_buffer("inv_freq", rotary_inv_freq(self.dim), persistent=False)

    def _heads(self, h, positions):
        x = self.norm(h)
        q, k, v = self.qkv(x).unflatten(-1, (3, self.heads, self.dim)).unbind(-3)
        q, k = qk_norm_rope(q, k, self.q_weight, self.k_weight, self.inv_freq, positions)
        g = F.logsigmoid(self.gate(x).float() + 4.0).to(x.dtype)
        return q, k, v, g.unflatten(-1, (self.heads, self.dim))

    def forward(self, h, positions, cu=None, keep=False):
        q, k, v, g = self._heads(h, positions)
        o, state = chunk_gla(q, k, v.contiguous(), g, output_final_state=keep, cu_seqlens=cu,
                             chunk_size=64)
        return h + self.out_proj(o.flatten(-2)), state

    def empty_pool(self, slots, like):
        return torch.zeros(slots, self.heads, self.dim, self.dim, device=like.device)

    def step(self, h, positions, pool, slots):
        q, k, v, g = self._heads(h[:, None], positions[:, None])
        o, state = fused_recurrent_gla(q, k, v.contiguous(), gk=g, initial_state=pool[slots.long()],
                                       output_final_state=True)
        pool[slots.long()] = state
        return h + self.out_proj(o[:, 0].flatten(-2))


class HybridLM(nn.Module):
    def __init__(self, vocab=64, width=256, heads=4):
        super().__init__()
        self.embed = nn.Embedding(vocab, width)
        self.ssm = SelectiveBlock(width, 2 * width)
        self.attention = AttentionBlock(width, heads)
        self.norm = nn.RMSNorm(width)
        self.head = nn.Linear(width, vocab, bias=False)

    def forward(self, tokens, positions=None, cu=None, keep=False):
        h, ssm = self.ssm(self.embed(tokens), cu, keep)
        h, att = self.attention(h, positions, cu, keep)
        return self.head(self.norm(h)), (ssm, att)

    @torch.no_grad()
    def prefill(self, prompts, pools, slots):
        """Runs the prompts (lists of tokens) packed into one row and keeps their states in
        `slots` of the pools; returns the last logits of each."""
        cu = [0]
        for p in prompts:
            cu.append(cu[-1] + len(p))
        dev = self.embed.weight.device
        tokens = torch.tensor([t for p in prompts for t in p], device=dev)[None]
        logits, ((window, state), att) = self(tokens, positions_of(cu, dev), cu, True)
        at = slots.long()
        pools[0][0][at], pools[0][1][at], pools[1][at] = window, state, att
        return logits[0, torch.tensor(cu[1:], device=dev) - 1]

    def empty_pools(self, slots):
        like = self.embed.weight
        return self.ssm.empty_pool(slots, like), self.attention.empty_pool(slots, like)

    @torch.no_grad()
    def step(self, tokens, positions, pools, slots):
        """The next token of each sequence: tokens and positions [B]."""
        h = self.ssm.step(self.embed(tokens), pools[0], slots)
        h = self.attention.step(h, positions, pools[1], slots)
        return self.head(self.norm(h))


def batch(gen, B, n, vocab, device):
    """Symbols, a separator (token 0), the symbols again; and which positions count."""
    s = torch.randint(1, vocab, (B, n), generator=gen)
    return torch.cat([s, torch.zeros(B, 1, dtype=torch.long), s], 1).to(device)


def train(model, steps, device, seed=0, report=print):
    gen = torch.Generator().manual_seed(seed)
    opt = torch.optim.AdamW(model.parameters(), lr=1e-3)
    losses = []
    for i in range(steps):
        n = int(torch.randint(4, 25, (1,), generator=gen))
        x = batch(gen, 32, n, model.embed.num_embeddings, device)
        logits, _ = model(x[:, :-1])
        loss = F.cross_entropy(logits[:, n:].float().flatten(0, 1), x[:, n + 1:].flatten())
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if (i + 1) % 100 == 0:
            report(f"step {i + 1}: loss {losses[-1].item():.3f}")
    return losses


def generate(model, prompts, new, slots=None):
    """Greedy continuation of packed prompts, `new` tokens each."""
    dev = model.embed.weight.device
    slots = torch.arange(len(prompts), dtype=torch.int32, device=dev) if slots is None else slots
    pools = model.empty_pools(int(slots.max()) + 1)
    token = model.prefill(prompts, pools, slots).argmax(-1)
    pos = torch.tensor([len(p) for p in prompts], device=dev)
    out = [token]
    for _ in range(new - 1):
        token = model.step(token, pos, pools, slots).argmax(-1)
        pos = pos + 1
        out.append(token)
    return torch.stack(out, 1)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=1000)
    args = ap.parse_args()
    torch.manual_seed(0)
    dev = torch.device("cuda:0")
    model = HybridLM().to(dev)
    train(model, args.steps, dev)
    gen = torch.Generator().manual_seed(1)
    symbols = [torch.randint(1, 64, (n,), generator=gen).tolist() for n in (5, 24, 12)]
    out = generate(model, [s + [0] for s in symbols], 24)
    for s, o in zip(symbols, out.tolist()):
        hit = sum(a == b for a, b in zip(s, o))
        print(f"{len(s)} symbols: {hit} copied")


if __name__ == "__main__":
    main()
