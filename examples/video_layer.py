"""The attention part of a video transformer's layer on htrc_b200's operators, and a few training steps of its prompt
branch (synthetic latents, states and weights).

    python examples/video_layer.py [--grid 16,32,32] [--heads 24] [--keys 256] [--train 0]

Self attention: q and k are normalised per head, turned by their (time, height, width) positions and laid out head by
head in one pass (``rotary_qk``), then attend through the flat operator (``flat_attention_heads``).  Cross attention:
the tokens read the states of an encoder, each batch entry its own number of them (``cross_attention``).  ``--train``
trains the prompt branch alone, as an adapter would: its gradients run through ``rotary_axes`` (the query norm, no
rotation) and ``cross_attention``.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import htrc_b200  # noqa: E402

AXES = (44, 42, 42)              # of a head's 128 elements: time, height, width


class SelfBranch(nn.Module):
    """Flat self attention of a latent grid's tokens (inference: the flat operator has no backward)."""

    def __init__(self, width, heads, exact_leaves):
        super().__init__()
        self.heads = heads
        self.cfg = {**htrc_b200.PROD, "leaf": 64, "exact_leaves": exact_leaves}
        self.qkv = nn.Linear(width, 3 * heads * 128, bias=False)
        self.out = nn.Linear(heads * 128, width, bias=False)
        self.norm = nn.ParameterList(nn.Parameter(torch.ones(128)) for _ in range(2))

    @torch.no_grad()
    def forward(self, x, positions):
        q, k, v = self.qkv(x).unflatten(-1, (3, self.heads, 128)).unbind(-3)       # strided views, no copies
        q, k = htrc_b200.rotary_qk(q, k, positions, axes=AXES, q_weight=self.norm[0], k_weight=self.norm[1],
                                   heads_first=True)
        a = torch.stack([htrc_b200.flat_attention_heads(*rows, **self.cfg)
                         for rows in zip(q, k, v.transpose(1, 2).contiguous())])    # [batch, heads, tokens, 128]
        return self.out(a.transpose(1, 2).flatten(2).to(x.dtype))


class PromptBranch(nn.Module):
    """Cross attention to an encoder's states, kv_heads shared by the query heads."""

    def __init__(self, width, state_width, heads, kv_heads):
        super().__init__()
        self.heads, self.kv_heads = heads, kv_heads
        self.q = nn.Linear(width, heads * 128, bias=False)
        self.kv = nn.Linear(state_width, 2 * kv_heads * 128, bias=False)
        self.out = nn.Linear(heads * 128, width, bias=False)
        self.norm = nn.ParameterList(nn.Parameter(torch.ones(128)) for _ in range(2))

    def forward(self, x, states, lengths):
        q = self.q(x).unflatten(-1, (self.heads, 128))
        k, v = self.kv(states).unflatten(-1, (2, self.kv_heads, 128)).unbind(-3)
        q, k = (htrc_b200.rotary_axes(r, r.new_zeros(r.shape[:2] + (1,), dtype=torch.int32), axes=(0,), weight=w)
                for r, w in zip((q, k), self.norm))                                 # no axis is turned: the norm alone
        return self.out(htrc_b200.cross_attention(q, k, v, key_lengths=lengths).flatten(2))


class VideoLayer(nn.Module):
    def __init__(self, width=1024, state_width=768, heads=24, kv_heads=8, exact_leaves=64):
        super().__init__()
        self.own = SelfBranch(width, heads, exact_leaves)
        self.prompt = PromptBranch(width, state_width, heads, kv_heads)

    def forward(self, x, positions, states, lengths):
        x = x + self.own(x, positions)
        return x + self.prompt(x, states, lengths)


def make(grid, heads, kv_heads, keys, width=1024, state_width=768, batch=2, exact_leaves=64, seed=0):
    """(layer, x, positions, states, lengths) on the current device: a prompt and a shorter one per batch entry."""
    torch.manual_seed(seed)
    layer = VideoLayer(width, state_width, heads, kv_heads, exact_leaves).cuda().bfloat16()
    n = grid[0] * grid[1] * grid[2]
    x = torch.randn((batch, n, width), device="cuda").bfloat16()
    states = torch.randn((batch, keys, state_width), device="cuda").bfloat16()
    lengths = torch.linspace(keys, max(1, keys // 4), batch, device="cuda").int()
    positions = htrc_b200.grid_positions(grid).expand(batch, -1, -1)
    return layer, x, positions, states, lengths


def train(layer, x, positions, states, lengths, steps, rate=3e-4):
    """Losses of steps that fit the prompt branch to another branch's answers; the self branch stays as it is."""
    torch.manual_seed(1)
    with torch.no_grad():
        x = x + layer.own(x, positions)
        like = layer.prompt
        goal = PromptBranch(x.shape[-1], states.shape[-1], like.heads, like.kv_heads).cuda().bfloat16()(x, states, lengths)
    opt = torch.optim.Adam(layer.prompt.parameters(), lr=rate, eps=1e-6)
    losses = []
    for _ in range(steps):
        loss = (layer.prompt(x, states, lengths) - goal).float().pow(2).mean() / goal.float().pow(2).mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    return losses


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--grid", default="16,32,32")
    ap.add_argument("--heads", type=int, default=24)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--keys", type=int, default=256)
    ap.add_argument("--train", type=int, default=0, help="training steps of the prompt branch")
    a = ap.parse_args()
    grid = tuple(int(g) for g in a.grid.split(","))
    layer, *args = make(grid, a.heads, a.kv_heads, a.keys)
    with torch.no_grad():
        for _ in range(3):
            y = layer(*args)
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        y = layer(*args)
        end.record()
    torch.cuda.synchronize()
    htrc_b200.cross_status()
    print(f"{args[0].shape[0]} x {args[0].shape[1]} tokens: {start.elapsed_time(end):.2f} ms, "
          f"rms {float(y.float().pow(2).mean().sqrt()):.3f}")
    if a.train:
        losses = train(layer, *args, a.train)
        print("prompt branch, relative error:", " ".join(f"{x:.3f}" for x in losses))


if __name__ == "__main__":
    main()
