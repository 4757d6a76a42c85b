"""The block operators' definitions in float64 on the CPU, with bounds on rounding.

Bounds: u is the unit roundoff of the operands' type (2^-24, 2^-11, 2^-8) and e = 2^-24.  A sum
of n float32 products is within n e of the sum of their magnitudes whatever its order.  A result
is rounded once (u), and a product's operand that was computed (probabilities, ds) once more.
"""

import math

import torch

ROUNDOFF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E = 2.0 ** -24
# Below a type's least normal number a rounding's error is absolute.  An exponential below
# float32's is 0 (FLUSH: the most that a probability may lose so).
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}
FLUSH = 2.0 ** -126


def visible(blocks, queries, keys, block, lengths, causal):
    """[batch, kv_heads, queries, keys]: keys that each query sees."""
    batch, _, kv_heads, _ = blocks.shape
    see = torch.zeros(batch, kv_heads, queries, keys, dtype=torch.bool)
    place_of = torch.arange(keys)
    for b in range(batch):
        length = keys if lengths is None else int(lengths[b])
        for t in range(queries):
            place = length - queries + t
            last = -1 if place < 0 else place if causal else length - 1
            for h in range(kv_heads):
                ids = [int(i) for i in blocks[b, t, h] if 0 <= int(i) <= last // block]
                if last >= 0 and ids:
                    listed = torch.zeros((keys + block - 1) // block, dtype=torch.bool)
                    listed[ids] = True
                    see[b, h, t] = listed[place_of // block] & (place_of <= last)
    return see


class Attention:
    """out, lse and, with dout, dq, dk, dv in float64, and how far each element may be off."""

    def __init__(self, q, k, v, blocks, block, lengths=None, causal=True, scale=None, dout=None):
        u, tiny = ROUNDOFF[q.dtype], TINY[q.dtype]
        batch, queries, q_heads, dim = q.shape
        keys, kv_heads = k.shape[1], k.shape[2]
        group = q_heads // kv_heads
        scale = 1.0 / math.sqrt(dim) if scale is None else scale
        see = visible(blocks, queries, keys, block, lengths, causal)[:, :, None]
        some = see.any(-1, keepdim=True)
        wide = lambda x: x.double().transpose(1, 2)  # noqa: E731  [batch, heads, rows, dim]
        q4 = wide(q).reshape(batch, kv_heads, group, queries, dim)
        k4, v4 = wide(k)[:, :, None], wide(v)[:, :, None]
        used = see.any(-2).any(-2)[..., None]  # keys that nobody sees may hold anything
        k4, v4 = (torch.where(used[:, :, None], x, 0.0) for x in (k4, v4))
        x = torch.where(see, q4 @ k4.transpose(-1, -2) * scale, -math.inf)
        lse = torch.logsumexp(x, -1, keepdim=True)
        p = torch.where(see, torch.exp(x - torch.where(some, lse, 0.0)), 0.0)
        out = p @ v4
        # a score's error: the product's sum and the scaling; lse's: its terms'
        xe = (dim + 4) * E * abs(scale) * (q4.abs() @ k4.abs().transpose(-1, -2))
        xe = xe + 4 * E * torch.where(see, x.abs(), 0.0)
        worst = torch.where(see, xe, 0.0).amax(-1, keepdim=True)
        count = see.sum(-1, keepdim=True)
        lse_off = worst + (count + 8) * E + 4 * E * torch.where(some, lse, 0.0).abs()
        # a probability's relative error (twice the exponent's), and with the operand's rounding
        pe = 2 * (xe + lse_off) + 8 * E
        flushed = torch.where(see, FLUSH, 0.0)
        spread = (p * (pe + u + count * E) + flushed) @ v4.abs()
        out_off = spread + u * out.abs() + tiny

        def rows(x, heads):
            return x.reshape(batch, heads, -1, x.shape[-1]).transpose(1, 2)

        self.out, self.out_off = rows(out, q_heads), 1.01 * rows(out_off, q_heads)
        self.lse = rows(lse, q_heads)[..., 0]
        self.lse_off = 1.01 * rows(lse_off, q_heads)[..., 0]
        if dout is None:
            return
        d4 = wide(dout).reshape(batch, kv_heads, group, queries, dim)
        dp = d4 @ v4.transpose(-1, -2)
        delta = (d4 * out).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        # delta is summed from the rounded out; dp from exact operands
        dp_off = (dim + 1) * E * (d4.abs() @ v4.abs().transpose(-1, -2))
        delta_off = (d4.abs() * (out_off + (dim + 1) * E * out.abs())).sum(-1, keepdim=True)
        ds_off = p * (pe * (dp - delta).abs() + dp_off + delta_off) + u * ds.abs()
        ds_off = ds_off + flushed * (dp - delta).abs()
        ds_off = torch.where(see, ds_off + 4 * E * ds.abs() + tiny, 0.0)
        n = count + 8
        dq = scale * (ds @ k4)
        dq_off = abs(scale) * ((ds_off + n * E * ds.abs()) @ k4.abs()) + u * dq.abs() + tiny
        each = see.sum(-2, keepdim=True).transpose(-1, -2) * group + 8  # queries of a key
        dk = scale * (ds.transpose(-1, -2) @ q4).sum(2)
        dk_off = (ds_off.transpose(-1, -2) @ q4.abs() +
                  each * E * (ds.abs().transpose(-1, -2) @ q4.abs())).sum(2) * abs(scale)
        dv = (p.transpose(-1, -2) @ d4).sum(2)
        p_off = torch.where(see, p * (pe + u) + tiny + FLUSH, 0.0)
        dv_off = (p_off.transpose(-1, -2) @ d4.abs() +
                  each * E * (p.transpose(-1, -2) @ d4.abs())).sum(2)
        self.dq, self.dq_off = rows(dq, q_heads), 1.01 * rows(dq_off, q_heads)
        self.dk, self.dk_off = rows(dk, kv_heads), 1.01 * rows(dk_off + u * dk.abs() + tiny,
                                                               kv_heads)
        self.dv, self.dv_off = rows(dv, kv_heads), 1.01 * rows(dv_off + u * dv.abs() + tiny,
                                                               kv_heads)


def near(got, want, off, what=""):
    """Every element within its bound, and infinities where the reference has them."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine], want[~fine]), what
    over = (got - want).abs()[fine] - off.expand_as(want)[fine]
    assert not torch.isnan(over).any(), f"{what}: NaN"
    assert over.numel() == 0 or float(over.max()) <= 0.0, \
        f"{what}: {float(over.max())} past its bound at {int(over.argmax())} of {over.numel()}"


def means(k, block, lengths=None):
    batch, keys, heads, dim = k.shape
    n = (keys + block - 1) // block
    out = torch.zeros(batch, n, heads, dim, dtype=torch.float64)
    size = torch.zeros_like(out)
    for b in range(batch):
        length = keys if lengths is None else int(lengths[b])
        for j in range(n):
            rows = k[b, j * block:min(length, (j + 1) * block)].double()
            if len(rows):
                out[b, j], size[b, j] = rows.mean(0), rows.abs().mean(0)
    return out, (block + 2) * E * size


def scores(q, mean, block, keys, lengths=None, causal=True, scale=None):
    batch, queries, q_heads, dim = q.shape
    kv_heads, n = mean.shape[2], mean.shape[1]
    group = q_heads // kv_heads
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    heads = q.double().reshape(batch, queries, kv_heads, group, dim)
    m = mean.double().permute(0, 2, 3, 1)
    x = (heads.sum(3).transpose(1, 2) @ m).transpose(1, 2) * scale
    off = (heads.abs().sum(3).transpose(1, 2) @ m.abs()).transpose(1, 2)
    off = (dim + group + 4) * E * abs(scale) * off
    first = torch.arange(n) * block
    for b in range(batch):
        length = keys if lengths is None else int(lengths[b])
        for t in range(queries):
            place = length - queries + t
            last = -1 if place < 0 else place if causal else length - 1
            x[b, t, :, first > last] = -math.inf
    return x, off


def select(score, count, block, keys, lengths=None, causal=True, sink=1, local=1):
    batch, queries, heads, n = score.shape
    ids = torch.full((batch, queries, heads, count), -1, dtype=torch.int32)
    for b in range(batch):
        length = keys if lengths is None else int(lengths[b])
        for t in range(queries):
            place = length - queries + t
            if place < 0:
                continue
            own = (place if causal else length - 1) // block
            first = [own - i for i in range(local) if own - i >= 0]
            first += [j for j in range(min(sink, own + 1)) if j not in first]
            for h in range(heads):
                row = score[b, t, h].double().tolist()
                rest = [j for j in range(own + 1) if j not in first and row[j] > -math.inf]
                rest.sort(key=lambda j: (-row[j], j))
                taken = sorted((first + rest)[:count])
                ids[b, t, h, :len(taken)] = torch.tensor(taken, dtype=torch.int32)
    return ids
