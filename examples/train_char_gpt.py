"""A small character-level GPT trained with sparse layers, end to end on one GPU.

    python examples/train_char_gpt.py [--steps 300] [--state-bits 8] [--act-bits 8]
                                      [--buckets 16] [--no-set]

Every projection is a SparseLinear; what stands between them is residual_norm, attention and
an activation (feature-major, as the sparse layers give and take it), the head and its loss are
linear_cross_entropy, the optimizer is AdamW, and SET rewires the sparse layers every few
steps while AdamW's moments follow their weights (``model.apply(opt.attach)``).
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
import torch.nn as nn

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import sparsecore_amd as slk  # noqa: E402


class Block(nn.Module):
    """Attention and feed-forward part; takes and returns the residual stream and the
    branch that is not yet added to it."""

    def __init__(self, d: int, heads: int, f: int, attn_sparsity: float, ffn_sparsity: float,
                 act_bits: int = 32):
        super().__init__()
        self.heads, self.act_bits = heads, act_bits
        self.norm1, self.norm2 = slk.ResidualNorm(d), slk.ResidualNorm(d)
        self.qkv = slk.SparseLinear(d, 3 * d, sparsity=attn_sparsity, bias=False,
                                    save_bits=act_bits)
        self.out = slk.SparseLinear(d, d, sparsity=attn_sparsity, bias=False,
                                    save_bits=act_bits)
        self.up = slk.SparseLinear(d, f, sparsity=ffn_sparsity, bias=False,
                                     save_bits=act_bits)
        self.down = slk.SparseLinear(f, d, sparsity=ffn_sparsity, bias=False,
                                     save_bits=act_bits)

    def forward(self, x, branch, rel=None):
        x, y = self.norm1(x, branch)
        q, k, v = (z.unflatten(-1, (self.heads, -1)) for z in self.qkv(y).chunk(3, dim=-1))
        a = slk.attention(q, k, v, bias=rel, max_distance=64, feature_major=True)
        x, y = self.norm2(x, self.out(a.flatten(2)))
        return x, self.down(slk.activation(self.up(y), "gelu", save_bits=self.act_bits))


class CharGPT(nn.Module):
    def __init__(self, vocab: int, ctx: int, d: int = 128, heads: int = 4, layers: int = 2,
                 attn_sparsity: float = 0.7, ffn_sparsity: float = 0.9, act_bits: int = 32,
                 buckets: int = 0):
        super().__init__()
        self.tok, self.pos = nn.Embedding(vocab, d), nn.Embedding(ctx, d)
        # learned biases of the relative position, shared by the blocks
        self.rel = nn.Parameter(torch.zeros(buckets, heads)) if buckets else None
        self.blocks = nn.ModuleList(Block(d, heads, 4 * d, attn_sparsity, ffn_sparsity, act_bits)
                                    for _ in range(layers))
        self.norm = slk.ResidualNorm(d, feature_major=False)
        self.head = nn.Parameter(torch.randn(vocab, d) * d ** -0.5)

    def forward(self, idx, target):
        x = self.tok(idx) + self.pos(torch.arange(idx.shape[1], device=idx.device))
        branch = None
        for block in self.blocks:
            x, branch = block(x, branch, self.rel)
        _, y = self.norm(x, branch)
        return slk.linear_cross_entropy(y, self.head, target)


def batches(text: str, ctx: int, batch: int, device, seed: int):
    """Random windows of the text and the characters that follow them."""
    chars = sorted(set(text))
    data = torch.tensor([chars.index(c) for c in text], device=device)
    gen = torch.Generator().manual_seed(seed)
    while True:
        at = torch.randint(0, len(data) - ctx - 1, (batch,), generator=gen).to(device)
        window = data[at[:, None] + torch.arange(ctx + 1, device=device)]
        yield window[:, :-1].contiguous(), window[:, 1:].contiguous()


def train(steps: int = 300, state_bits: int = 32, rewire: bool = True, seed: int = 0,
          log=None, act_bits: int = 32, buckets: int = 0) -> list[float]:
    """Trains on this file's own text; returns the loss of every step."""
    device, ctx = torch.device("cuda"), 64
    text = Path(__file__).read_text()
    torch.manual_seed(seed)
    model = CharGPT(len(set(text)), ctx, act_bits=act_bits, buckets=buckets).to(device)
    opt = slk.AdamW(model.parameters(), lr=2e-3, weight_decay=0.01, state_bits=state_bits)
    model.apply(opt.attach)
    algo = slk.SET(sparsity=0.9, drop_fraction=0.2, update_freq=50, seed=seed)
    if rewire:
        model.apply(algo)
    losses = []
    data = batches(text, ctx, 32, device, seed)
    for step in range(steps):
        idx, target = next(data)
        opt.zero_grad()
        loss = model(idx, target)
        loss.backward()
        opt.step()
        if rewire:
            algo.step()
        losses.append(loss.detach())
        if log is not None and (step % 50 == 0 or step + 1 == steps):
            log(f"step {step:4d}  loss {float(losses[-1]):.3f}")
    return [float(x) for x in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--state-bits", type=int, default=32, choices=(8, 32))
    ap.add_argument("--act-bits", type=int, default=32, choices=(8, 32),
                    help="of what the blocks keep for their backward")
    ap.add_argument("--buckets", type=int, default=0,
                    help="learn a bias of the relative position in so many buckets")
    ap.add_argument("--no-set", action="store_true", help="keep the initial connections")
    args = ap.parse_args()
    train(args.steps, args.state_bits, not args.no_set, log=print, act_bits=args.act_bits,
          buckets=args.buckets)
