"""The linear cross entropy and its gradients by their formulas in float64, and how far a result of
float32 sums and operands of 16 bits may be off.

Bounds: u is the unit roundoff of the operands' type (2^-24, 2^-11, 2^-8) and e = 2^-24.  A sum of n
float32 products is within n e of the sum of their magnitudes whatever its order.  A gradient's
products take dz rounded to the operands' type (u), 16-bit ones of up to 128 tokens in two parts
(u^2), and results are rounded once (u).
"""

import torch

ROUNDOFF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E = 2.0 ** -24
# Below a type's least normal number a rounding's error is absolute: half of the least step (all
# of it where float32 flushes to 0).  float16's dz is 2^14 dz.
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
DZ_TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -39, torch.bfloat16: 2.0 ** -126}


class Loss:
    """each (a token's loss), loss, lse and, with dloss, dx and dtable; x_off for how far x may be
    off.  Tokens without a target (outside the words) may hold anything."""

    def __init__(self, x, table, targets, scale=1.0, reduction="mean", dloss=None):
        u, tiny = ROUNDOFF[x.dtype], TINY[x.dtype]
        shape, width, words = x.shape, x.shape[-1], table.shape[0]
        x, targets = x.detach().reshape(-1, width), targets.reshape(-1).long()
        held = (targets >= 0) & (targets < words)
        at = torch.where(held, targets, 0)[:, None]
        n = int(held.sum())
        wide = torch.where(held[:, None], x, 0.0).double()
        w = table.detach().double()
        f32 = float(torch.tensor(scale, dtype=torch.float32))
        z = wide @ w.T * f32
        ze = (width + 2) * E * abs(f32) * (wide.abs() @ w.abs().T)
        top = z.amax(-1, keepdim=True)
        lse = torch.logsumexp(z, -1, keepdim=True)
        # an exponential's relative error: its argument's, and the function's own
        pe = 2 * (ze + ze.amax(-1, keepdim=True)) + 4 * E * (z - top).abs() + 8 * E
        p = torch.exp(z - lse)
        total_e = (p * pe).sum(-1, keepdim=True) + (words + 8) * E
        each = torch.where(held, (lse - z.gather(1, at))[:, 0], 0.0)
        # log's own error is relative to it and, near 1, to its argument
        each_off = (total_e + 4 * E * (1 + (lse - top).abs()) + 2 * E * (top - z.gather(1, at)).abs()
                    + ze.gather(1, at) + ze.amax(-1, keepdim=True))[:, 0]
        self.lse, self.lse_off = lse[:, 0], each_off + 2 * E * lse[:, 0].abs()
        each_off = torch.where(held, each_off, 0.0)
        self.each, self.each_off = each.view(shape[:-1]), each_off.view(shape[:-1])
        if reduction == "none":
            self.loss, self.loss_off = self.each, self.each_off
        else:
            count = max(n, 1) if reduction == "mean" else 1
            self.loss = each.sum() / count
            self.loss_off = each_off.sum() / count + 4 * E * self.loss.abs()
        if dloss is None:
            return
        c = dloss.detach().double().reshape(-1).expand(len(x))
        if reduction == "mean":
            c = c / max(n, 1)
        c = torch.where(held, c, 0.0)[:, None]
        one = torch.zeros_like(p).scatter_(1, at, 1.0)
        dz = (p - one) * c
        dz_u = u * u if len(x) <= 128 and x.dtype != torch.float32 else u
        off = (p * (pe + total_e) + 2 * E * one + 4 * E * (p - one).abs() +
               dz_u * (p - one).abs()) * c.abs() + DZ_TINY[x.dtype] * c.abs().amax()
        s = abs(f32)
        dx, dtable = dz @ w * f32, dz.T @ wide * f32
        dx_off = s * (off @ w.abs() + (words + 8) * E * (dz.abs() @ w.abs()))
        dtable_off = s * (off.T @ wide.abs() + (2 * n + 4) * E * (dz.abs().T @ wide.abs()))
        self.dx, self.dx_off = dx.view(shape), (dx_off + u * dx.abs() + tiny).view(shape)
        self.dtable, self.dtable_off = dtable, dtable_off + u * dtable.abs() + tiny


def near(got, want, off, what=""):
    assert got.shape == want.shape, what
    most = torch.finfo(got.dtype).max
    got = got.detach().double()
    # Rounding to the nearest makes an infinity of what is half a step past the type's largest
    # number or more; a value that may lie there may be either.
    past = (got == torch.inf * want.sign()) & (want.abs() + 1.01 * off >= most)
    over = (torch.where(past, want, got) - want).abs() - 1.01 * off
    assert not torch.isnan(over).any(), what
    assert over.numel() == 0 or float(over.max()) <= 0.0, f"{what}: {float(over.max())} past"
