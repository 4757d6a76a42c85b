"""One layer of a language model on computed sparsity: attention over selected blocks of keys, and
experts that tokens are routed to.  Trains on a synthetic task, then decodes with a cache.

    python -m nacho_amd.examples.block_layer [--steps 160]

The task: a random phrase, then blanks in which it is to be said again, twice.  A blank has to find
the token one or two phrases earlier, in a block that its score selects.
"""

from __future__ import annotations

import argparse

import torch
from torch import nn
from torch.nn import functional as F

import nacho_amd


class BlockAttention(nn.Module):
    """Each query attends to `count` blocks of `block` keys: the first, its own and the best."""

    def __init__(self, dim, q_heads, kv_heads, head_dim, block=32, count=4):
        super().__init__()
        self.sizes, self.block, self.count = (q_heads, kv_heads, head_dim), block, count
        self.qkv = nn.Linear(dim, (q_heads + 2 * kv_heads) * head_dim, bias=False)
        self.out = nn.Linear(q_heads * head_dim, dim, bias=False)

    def project(self, x):
        hq, hk, d = self.sizes
        qkv = self.qkv(x).unflatten(-1, (hq + 2 * hk, d))
        return qkv.split((hq, hk, hk), -2)  # views: the operators take their strides

    def attend(self, q, k, v, means, lengths=None):
        keys = k.shape[1]
        with torch.no_grad():  # the choice of blocks has no gradient
            scores = nacho_amd.gpu_block_scores(q, means, self.block, keys, lengths)
            blocks = nacho_amd.gpu_block_select(scores, self.count, self.block, keys, lengths)
        out = nacho_amd.gpu_block_attention(q, k, v, blocks, self.block, lengths)
        return self.out(out.flatten(-2))

    def forward(self, x):
        q, k, v = self.project(x)
        return self.attend(q, k, v, nacho_amd.gpu_block_means(k.detach(), self.block))


class Experts(nn.Module):
    """Each token goes to `per_token` of the experts; their outputs come back weighted."""

    def __init__(self, dim, hidden, experts, per_token=2):
        super().__init__()
        self.per_token = per_token
        self.router = nn.Linear(dim, experts, bias=False)
        self.up = nn.Parameter(torch.randn(experts, dim, hidden) * dim ** -0.5)
        self.down = nn.Parameter(torch.randn(experts, hidden, dim) * hidden ** -0.5)

    def forward(self, x):
        tokens = x.reshape(-1, x.shape[-1])
        top, experts = torch.topk(self.router(tokens).float(), self.per_token, -1)
        route = nacho_amd.gpu_route(experts, self.up.shape[0])
        rows = nacho_amd.gpu_dispatch(tokens, route)
        # the experts' products: each has the rows between its offsets
        ends = route.pos.tolist()
        parts = [F.gelu(rows[a:b] @ up) @ down
                 for a, b, up, down in zip(ends, ends[1:], self.up, self.down)]
        out = nacho_amd.gpu_combine(torch.cat(parts), route, torch.softmax(top, -1))
        return out.view_as(x)


class Layer(nn.Module):
    def __init__(self, words, dim=128, q_heads=8, kv_heads=2, head_dim=64, hidden=128, experts=4):
        super().__init__()
        self.words = nn.Embedding(words, dim)
        self.attention = BlockAttention(dim, q_heads, kv_heads, head_dim)
        self.experts = Experts(dim, hidden, experts)
        self.norms = nn.ModuleList(nn.LayerNorm(dim) for _ in range(3))
        self.head = nn.Linear(dim, words, bias=False)

    def rest(self, x, attended):
        x = x + attended
        x = x + self.experts(self.norms[1](x))
        return self.head(self.norms[2](x))

    def forward(self, tokens, places):
        x = self.words(tokens) + places[:tokens.shape[1]]
        return self.rest(x, self.attention(self.norms[0](x)))


class Cache:
    """Keys, values and block means of a batch of sequences that grow token by token."""

    def __init__(self, batch, keys, layer, like):
        hq, hk, d = layer.attention.sizes
        self.k, self.v = (like.new_zeros(batch, keys, hk, d) for _ in range(2))
        blocks = -(-keys // layer.attention.block)
        self.means = torch.zeros(batch, blocks, hk, d, device=like.device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=like.device)


def decode(layer, cache, token, place):
    """Logits of one more token of each sequence, [batch, 1, words]."""
    attention = layer.attention
    x = layer.words(token) + place
    q, k, v = attention.project(layer.norms[0](x))
    at = int(cache.lengths[0])
    cache.k[:, at], cache.v[:, at] = k[:, 0], v[:, 0]
    cache.lengths += 1
    # the newest block's mean is all that a token changes
    first = at // attention.block * attention.block
    mine = cache.k[:, first:first + attention.block]
    cache.means[:, at // attention.block] = nacho_amd.gpu_block_means(
        mine, attention.block, cache.lengths - first)[:, 0]
    return layer.rest(x, attention.attend(q, cache.k, cache.v, cache.means, cache.lengths))


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--steps", type=int, default=160)
    args = parser.parse_args(argv)
    torch.manual_seed(0)
    device, words, phrase, length, batch = torch.device("cuda"), 64, 96, 288, 8
    # A place has the code of the place a phrase later.
    turns = torch.arange(length, device=device)[:, None] * torch.arange(1, 65, device=device)
    turns = turns * (2 * torch.pi / phrase)
    places = torch.cat((turns.sin(), turns.cos()), -1)
    layer = Layer(words).to(device)
    optimiser = torch.optim.Adam(layer.parameters(), lr=3e-3)

    def sequences():
        said = torch.randint(1, words, (batch, phrase), device=device)
        blanks = torch.zeros(batch, length - phrase, dtype=torch.long, device=device)
        return torch.cat((said, blanks), 1), said.repeat(1, length // phrase)

    losses = []
    for step in range(args.steps):
        tokens, wanted = sequences()
        logits = layer(tokens, places)
        loss = F.cross_entropy(logits[:, phrase:].flatten(0, 1), wanted[:, phrase:].flatten())
        optimiser.zero_grad()
        loss.backward()
        optimiser.step()
        losses.append(float(loss.detach()))
        if step % 20 == 0 or step + 1 == args.steps:
            print(f"step {step:4d}  loss {losses[-1]:.3f}", flush=True)

    with torch.no_grad():
        tokens = sequences()[0][:2]
        whole = layer(tokens, places)
        cache = Cache(2, length, layer, whole)
        apart = 0.0
        for t in range(length):
            logits = decode(layer, cache, tokens[:, t:t + 1], places[t])
            apart = max(apart, float((logits[:, 0] - whole[:, t]).abs().max()))
    print(f"decoded {length} tokens of 2 sequences: logits at most {apart:.2g} from the whole pass",
          flush=True)
    return losses, apart


if __name__ == "__main__":
    main()
