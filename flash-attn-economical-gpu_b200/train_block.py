"""A small decoder that trains on the operators of `training`: packed sequences through pre-norm blocks of layer norm
with the residual add, rotary embedding with three position axes, and packed causal attention, with their gradients.

    python train_block.py --steps 50            # prints the loss and the time of a step

The data is synthetic: sequences of one "text" run and one "image" of height x width patches, filled with one of a few
fixed words over and over.  Most tokens occur in several words, so the next token follows from the tokens before.  Text tokens advance all
three axes together; an image's patches share a time and differ in height and width.  Projections, GELU and the cross
entropy are PyTorch's.  No counterpart in the reference, which has no backward pass.
"""
from __future__ import annotations

import argparse
import time

import torch
import torch.nn.functional as F

import training


class Block(torch.nn.Module):
    """x, branch -> x, branch: each norm adds the previous branch to the stream as it reads it."""

    def __init__(self, width: int, heads: int, heads_kv: int, head_dim: int):
        super().__init__()
        self.heads, self.heads_kv, self.head_dim = heads, heads_kv, head_dim
        self.norm1, self.bias1 = torch.nn.Parameter(torch.ones(width)), torch.nn.Parameter(torch.zeros(width))
        self.norm2, self.bias2 = torch.nn.Parameter(torch.ones(width)), torch.nn.Parameter(torch.zeros(width))
        self.qkv = torch.nn.Linear(width, (heads + 2 * heads_kv) * head_dim, bias=False, dtype=torch.bfloat16)
        self.proj = torch.nn.Linear(heads * head_dim, width, bias=False, dtype=torch.bfloat16)
        self.up = torch.nn.Linear(width, 4 * width, bias=False, dtype=torch.bfloat16)
        self.down = torch.nn.Linear(4 * width, width, bias=False, dtype=torch.bfloat16)

    def forward(self, x, branch, batch):
        h, x = training.layernorm(x, self.norm1, self.bias1, residual=branch)
        qkv = self.qkv(h).view(x.shape[0], self.heads + 2 * self.heads_kv, self.head_dim)
        q, k, v = qkv.split([self.heads, self.heads_kv, self.heads_kv], 1)
        q, k = training.rope(q, k, batch["positions"], batch["cos"], batch["sin"], batch["sections"])
        o = training.attention_varlen(q, k, v, batch["cu"], batch["cu"], batch["longest"], batch["longest"], causal=True)
        h, x = training.layernorm(x, self.norm2, self.bias2, residual=self.proj(o.flatten(1)))
        return x, self.down(F.gelu(self.up(h)))


class Decoder(torch.nn.Module):
    def __init__(self, vocab: int, width: int, layers: int, heads: int, heads_kv: int, head_dim: int):
        super().__init__()
        self.embed = torch.nn.Embedding(vocab, width, dtype=torch.bfloat16)
        self.blocks = torch.nn.ModuleList(Block(width, heads, heads_kv, head_dim) for _ in range(layers))
        self.norm, self.bias = torch.nn.Parameter(torch.ones(width)), torch.nn.Parameter(torch.zeros(width))
        self.head = torch.nn.Linear(width, vocab, bias=False, dtype=torch.bfloat16)

    def forward(self, tokens, batch):
        x = self.embed(tokens)
        branch = torch.zeros_like(x)
        for block in self.blocks:
            x, branch = block(x, branch, batch)
        h, _ = training.layernorm(x, self.norm, self.bias, residual=branch)
        return self.head(h)


def rope_positions(text: int, height: int, width: int) -> torch.Tensor:
    """[3, text + height * width]: (time, height, width) of a text run followed by one image."""
    run = torch.arange(text).expand(3, -1)
    h, w = torch.meshgrid(torch.arange(height), torch.arange(width), indexing="ij")
    image = torch.stack((torch.zeros(height * width, dtype=torch.long), h.flatten(), w.flatten())) + text
    return torch.cat((run, image), 1)


def make_batch(shapes, words, sections, generator, device):
    """A packed batch of sequences given as (text tokens, image height, image width), each one of `words` repeated."""
    tokens, positions, lengths = [], [], []
    for text, height, width in shapes:
        n = text + height * width
        word = words[int(torch.randint(0, len(words), (), generator=generator))]
        tokens.append(word.repeat(n // len(word) + 1)[:n])
        positions.append(rope_positions(text, height, width))
        lengths.append(n)
    positions = torch.cat(positions, 1).to(device)
    half = sum(sections)
    angles = torch.arange(int(positions.max()) + 1, device=device)[:, None] * 10000.0 ** (
        -torch.arange(half, device=device) / half)
    cu = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device=device)
    return torch.cat(tokens).to(device), {"positions": positions, "cos": angles.cos(), "sin": angles.sin(),
                                          "sections": sections, "cu": cu, "longest": max(lengths)}


def next_token_loss(logits, tokens, cu):
    """Mean cross entropy of the next token, over all tokens that have one in their sequence."""
    has_next = torch.ones(tokens.numel(), dtype=torch.bool, device=tokens.device)
    has_next[cu[1:].long() - 1] = False
    targets = tokens.roll(-1)
    return F.cross_entropy(logits.float()[has_next], targets[has_next])


def train(steps: int, *, vocab=64, words=16, width=512, layers=2, heads=8, heads_kv=2, head_dim=64, sections=(8, 12, 12),
          shapes=((40, 14, 9), (3, 20, 20), (257, 4, 6), (1, 8, 8)), lr=2e-3, seed=0, device="cuda", log=None):
    """The loss of every step."""
    torch.manual_seed(seed)
    generator = torch.Generator().manual_seed(seed)
    model = Decoder(vocab, width, layers, heads, heads_kv, head_dim).to(device)
    words = torch.randint(0, vocab, (words, 7), generator=generator)
    optimizer = torch.optim.AdamW(model.parameters(), lr=lr)
    losses = []
    for step in range(steps):
        tokens, batch = make_batch(shapes, words, sections, generator, device)
        start = time.perf_counter()
        loss = next_token_loss(model(tokens, batch), tokens, batch["cu"])
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
        if log:
            log(f"step {step}: loss {losses[-1]:.3f}, {1e3 * (time.perf_counter() - start):.1f} ms")
    return losses


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=50)
    train(parser.parse_args().steps, log=print)
