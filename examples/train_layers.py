"""Trains a small language model with the package's operators around its optimizer: residual_norm between the blocks (post
norm, dropout, gate, residual add and the next pre norm in one pass), dropout on the embeddings, linear_cross_entropy on
the hidden states and the head's weight, and KronWhiten on the gradients. The text is a synthetic sequence in which nine
tokens of ten follow from the one before, so the loss can fall from log(vocabulary) to about a tenth of it.

    python examples/train_layers.py [--steps 200] [--dtype bf16|fp32]
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from psgd_pro_b200 import KronWhiten, layers  # noqa: E402


class Block(torch.nn.Module):
    """A feed-forward block on a token and the one before it, and the parameters of the joint after it."""

    def __init__(self, d, hidden, dtype):
        super().__init__()
        make = lambda *s: torch.nn.Parameter((torch.randn(*s) / math.sqrt(s[-1])).to("cuda", dtype))  # noqa: E731
        self.up, self.down = make(hidden, 2 * d), make(d, hidden)
        self.post, self.pre = (torch.nn.Parameter(torch.ones(d, device="cuda", dtype=dtype)) for _ in range(2))
        self.gate = torch.nn.Parameter(torch.full((d,), 0.5, device="cuda", dtype=dtype))

    def forward(self, x):
        before = torch.nn.functional.pad(x[:, :-1], (0, 0, 1, 0))
        return torch.relu(torch.cat([x, before], dim=-1) @ self.up.t()) @ self.down.t()


class Model(torch.nn.Module):
    def __init__(self, vocabulary=257, d=128, hidden=512, blocks=3, dropout=0.1, dtype=torch.bfloat16, seed=0):
        super().__init__()
        torch.manual_seed(seed)
        self.embed = torch.nn.Parameter((torch.randn(vocabulary, d) * 0.5).to("cuda", dtype))
        self.head = torch.nn.Parameter((torch.randn(vocabulary, d) / math.sqrt(d)).to("cuda", dtype))
        self.first = torch.nn.Parameter(torch.ones(d, device="cuda", dtype=dtype))
        self.blocks = torch.nn.ModuleList(Block(d, hidden, dtype) for _ in range(blocks))
        self.dropout, self.seed = dropout, seed

    def forward(self, tokens, target, step):
        """The mean loss of the tokens whose target is not -100. Every use of dropout has an offset of its own."""
        p, uses = self.dropout if self.training else 0.0, len(self.blocks) + 1
        x = self.embed[tokens]
        if p:
            x = layers.dropout(x, p, self.seed, step * uses)
        x, normed = layers.residual_norm(x, torch.zeros_like(x), weight=self.first)  # the first block's pre norm
        for k, block in enumerate(self.blocks):
            x, normed = layers.residual_norm(x, block(normed), post_norm=True, weight=block.pre, post_weight=block.post,
                                             gate=block.gate, dropout_p=p, seed=self.seed, offset=step * uses + k + 1)
        return layers.linear_cross_entropy(normed, self.head, target)


def batch(vocabulary, rows, length, generator):
    t = torch.randint(0, vocabulary, (rows, length + 1), generator=generator)
    follows = torch.rand(rows, length + 1, generator=generator) < 0.9
    for i in range(1, length + 1):
        t[:, i] = torch.where(follows[:, i], (3 * t[:, i - 1] + 7) % vocabulary, t[:, i])
    target = t[:, 1:].clone()
    target[:, -1] = -100  # the end of the text counts as padding
    return t[:, :-1].cuda(), target.cuda()


def train(steps=200, dtype=torch.bfloat16, vocabulary=257, rows=32, length=64, dropout=0.05, every=20, say=print):
    """The mean losses of the first and the last ten steps."""
    model = Model(vocabulary, dropout=dropout, dtype=dtype)
    opt = KronWhiten(list(model.parameters()), preconditioner_init_scale=1.0, lr_params=2e-3, momentum=0.9)
    g, losses = torch.Generator().manual_seed(1), []
    for step in range(steps):
        tokens, target = batch(vocabulary, rows, length, g)
        losses.append(opt.step(lambda: model(tokens, target, step)).item())
        if step % every == 0 or step == steps - 1:
            say(f"step {step:4d}  loss {losses[-1]:.4f}")
    opt.check_errors()
    layers.check_errors()
    return sum(losses[:10]) / 10, sum(losses[-10:]) / 10


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--dtype", choices=("bf16", "fp32"), default="bf16")
    a = ap.parse_args()
    train(a.steps, {"bf16": torch.bfloat16, "fp32": torch.float32}[a.dtype])
