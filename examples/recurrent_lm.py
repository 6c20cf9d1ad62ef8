"""A small recurrent language model on the operators of linrec_amd: trained on sequences whose next token follows from the last
two, then served, the prompts packed side by side and one token at a time from there.

    python examples/recurrent_lm.py [--steps 200] [--dtype f32|bf16]
"""
import argparse
import math
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import linrec_amd  # noqa: E402


class Block(nn.Module):
    """x + project(norm(gated recurrence of three projections of norm(x)))"""

    def __init__(self, width, heads):
        super().__init__()
        self.heads = heads
        self.before, self.before_bias = nn.Parameter(torch.ones(width)), nn.Parameter(torch.zeros(width))
        self.after, self.after_bias = nn.Parameter(torch.ones(width)), nn.Parameter(torch.zeros(width))
        self.into = nn.Linear(width, 3 * width)
        self.out = nn.Linear(width, width)
        # decays from 0.9 to 0.999 where the gate is wide open
        self.rate = nn.Parameter(torch.log(torch.expm1(-torch.log(torch.linspace(0.9, 0.999, width)) / 8.0)))

    def _project(self, x):
        normed = linrec_amd.group_norm_act(x.reshape(-1, x.shape[-1]), 1, self.before, self.before_bias, act="none")
        return self.into(normed).view(*x.shape[:-1], -1).chunk(3, -1)

    def _leave(self, x, h):
        normed = linrec_amd.group_norm_act(h.reshape(-1, h.shape[-1]), self.heads, self.after, self.after_bias, act="silu")
        return x + self.out(normed).view(x.shape)

    def forward(self, x, state=None, cu_seqlens=None):
        h, state = linrec_amd.gated_linrec(*self._project(x), self.rate, h0=state, cu_seqlens=cu_seqlens, return_state=True)
        return self._leave(x, h), state

    def step(self, x, state, slots):
        return self._leave(x, linrec_amd.gated_linrec_step(*self._project(x), self.rate, state, slots=slots))


class RecurrentLM(nn.Module):
    def __init__(self, vocab, width, heads, layers, dtype=torch.float32):
        super().__init__()
        self.scale = math.sqrt(width)
        self.table = nn.Parameter(torch.randn(vocab, width) / self.scale)
        self.blocks = nn.ModuleList(Block(width, heads) for _ in range(layers))
        self.norm, self.norm_bias = nn.Parameter(torch.ones(width)), nn.Parameter(torch.zeros(width))
        self.head = nn.Linear(width, vocab)
        self.to(dtype)
        for block in self.blocks:  # rates and the norms' parameters stay in 32 bits
            for name in ("rate", "before", "before_bias", "after", "after_bias"):
                getattr(block, name).data = getattr(block, name).data.float()
        self.norm.data, self.norm_bias.data = self.norm.data.float(), self.norm_bias.data.float()

    def _logits(self, x):
        normed = linrec_amd.group_norm_act(x.reshape(-1, x.shape[-1]), 1, self.norm, self.norm_bias, act="none")
        return self.head(normed).view(*x.shape[:-1], -1)

    def forward(self, tokens):
        """Logits of (batch, time) tokens."""
        x = linrec_amd.embedding(tokens, self.table, scale=self.scale)
        for block in self.blocks:
            x, _ = block(x)
        return self._logits(x)

    @torch.no_grad()
    def prefill(self, tokens, cu_seqlens, cache, slots):
        """Logits behind the last token of every packed prompt; the prompts' states go to rows `slots` of the layers' caches."""
        x = linrec_amd.embedding(tokens, self.table, scale=self.scale)
        for block, states in zip(self.blocks, cache):
            x, state = block(x, cu_seqlens=cu_seqlens)
            states[slots.long()] = state
        return self._logits(x[cu_seqlens[1:].long() - 1])

    @torch.no_grad()
    def step(self, tokens, cache, slots):
        """Logits behind one token of every running request."""
        x = linrec_amd.embedding(tokens, self.table, scale=self.scale)
        for block, states in zip(self.blocks, cache):
            x = block.step(x, states, slots)
        return self._logits(x)

    def new_cache(self, rows):
        width = self.table.shape[1]
        return [torch.zeros(rows, width, device=self.table.device) for _ in self.blocks]


def next_token(last, before, vocab):
    """One of two permutations of the vocabulary, by whether the token before the last was even."""
    return (last + torch.where(before % 2 == 0, 3, 10)) % vocab


def batch_of(batch, time, vocab, generator, device):
    tokens = list(torch.randint(0, vocab, (2, batch), generator=generator))
    while len(tokens) < time:
        tokens.append(next_token(tokens[-1], tokens[-2], vocab))
    return torch.stack(tokens, 1).to(device)


def train(model, steps, batch=32, time=64, lr=3e-3, seed=0):
    """Losses of the steps."""
    vocab, device = model.table.shape[0], model.table.device
    generator = torch.Generator().manual_seed(seed)
    optimizer = torch.optim.AdamW(model.parameters(), lr=lr)
    losses = []
    for _ in range(steps):
        tokens = batch_of(batch, time, vocab, generator, device)
        logits = model(tokens[:, :-1]).float()
        loss = nn.functional.cross_entropy(logits.reshape(-1, vocab), tokens[:, 1:].reshape(-1))
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return [float(v) for v in losses]


def serve(model, prompts, new_tokens):
    """Greedy continuations of `prompts` (lists of tokens)."""
    device = model.table.device
    rows = torch.randperm(2 * len(prompts))[:len(prompts)].to(device=device, dtype=torch.int32)
    cache = model.new_cache(2 * len(prompts))
    bounds = torch.tensor([0] + [len(p) for p in prompts]).cumsum(0).to(device=device, dtype=torch.int32)
    logits = model.prefill(torch.tensor(sum(prompts, []), device=device), bounds, cache, rows)
    out = []
    for _ in range(new_tokens):
        out.append(logits.argmax(-1))
        logits = model.step(out[-1], cache, rows)
    return torch.stack(out, 1)


def main():
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--dtype", choices=["f32", "bf16"], default="f32")
    args = parser.parse_args()
    torch.manual_seed(0)
    model = RecurrentLM(vocab=64, width=128, heads=4, layers=2, dtype=torch.bfloat16 if args.dtype == "bf16" else torch.float32).cuda()
    losses = train(model, args.steps)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} after {args.steps} steps")
    prompts = batch_of(3, 20, 64, torch.Generator().manual_seed(1), "cpu").tolist()
    prompts = [prompts[0], prompts[1][:9], prompts[2][:14]]
    for prompt, more in zip(prompts, serve(model, prompts, 10).tolist()):
        whole, right = prompt + more, 0
        for n in range(len(prompt), len(whole)):
            right += int(next_token(torch.tensor(whole[n - 1]), torch.tensor(whole[n - 2]), 64)) == whole[n]
        print(prompt[-4:], "->", more, f"({right} of {len(more)} as they should be)")


if __name__ == "__main__":
    main()
