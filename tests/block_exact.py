"""Block attention and its gradients by their formulas in float64, with what each query sees given
as a mask; and the comparison of a result with what rounding the exact one once leaves."""

import math

import torch


def attention(q, k, v, see, out=None, dout=None, scale=None):
    """out, or with dout (out, dq, dk, dv).  see: [batch, kv_heads, queries, keys].  delta is that
    of the given `out` (the backward pass's operand), or of the exact one."""
    batch, queries, q_heads, dim = q.shape
    kv_heads = k.shape[2]
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    shape = batch, kv_heads, q_heads // kv_heads, queries, dim

    def rows(x):
        return x.double().transpose(1, 2).reshape(shape)

    def back(x, heads):
        return x.reshape(batch, heads, -1, dim).transpose(1, 2)

    see = see[:, :, None]
    q4 = rows(q)
    k4, v4 = (x.double().transpose(1, 2)[:, :, None] for x in (k, v))
    x = torch.where(see, q4 @ k4.transpose(-1, -2) * scale, -math.inf)
    lse = torch.logsumexp(x, -1, keepdim=True)
    p = torch.where(see, torch.exp(x - lse), 0.0)
    o = p @ v4
    if dout is None:
        return back(o, q_heads)
    d4 = rows(dout)
    delta = (d4 * (o if out is None else rows(out))).sum(-1, keepdim=True)
    ds = torch.where(see, p * (d4 @ v4.transpose(-1, -2) - delta), 0.0) * scale
    return (back(o, q_heads), back(ds @ k4, q_heads),
            back((ds.transpose(-1, -2) @ q4).sum(2), kv_heads),
            back((p.transpose(-1, -2) @ d4).sum(2), kv_heads))


def rounded_once(got, want, what, share=1.02):
    """The result is off by no more than `share` of what rounding the exact one to its type is, in
    the 2-norm."""
    best = (want.to(got.dtype).double() - want).norm()
    off = (got.detach().double().cpu() - want).norm()
    assert math.isfinite(float(best)) and best > 0.0, what
    assert off <= share * best, f"{what}: {float(off / best):.3f} of rounding the exact one once"
