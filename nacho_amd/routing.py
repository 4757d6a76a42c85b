"""Tokens sorted by expert and back, with weights applied, and their gradients.

`gpu_route` turns a router's choices (experts of each token) into sparse structure, experts x
tokens; `gpu_dispatch` gathers the tokens' rows expert by expert, and `gpu_combine` brings the
experts' rows back, weighted and summed per token.  Both are differentiable through torch's
autograd, and every sum has a fixed order.

Calls are asynchronous on torch's current stream, read nothing back and may be captured in a
graph.  There is no CPU fallback.
"""

from __future__ import annotations

import torch

from .blocks import _TYPES, _call, _check_tensor, _device_of, _has_derivatives
from .tensors import CSR_gpu

MAX_EXPERTS = 2048


class Route:
    """A router's choices as structure.  The entry e = token * per_token + i is token's i-th
    choice; entries are sorted by expert, in order of e within one.

    pos    int32 [experts + 1]: expert x has the places pos[x] .. pos[x + 1]
    order  int32 [tokens * per_token]: the entry at each place; dropped entries behind
    slot   int32 [tokens, per_token]: the place of each entry, -1 for a dropped one
    """

    __slots__ = ("pos", "order", "slot", "tokens", "per_token", "experts")

    def __init__(self, pos, order, slot):
        self.pos, self.order, self.slot = pos, order, slot
        self.tokens, self.per_token = slot.shape
        self.experts = pos.numel() - 1

    def csr(self, weights: torch.Tensor) -> CSR_gpu:
        """The experts x tokens matrix of the weights [tokens, per_token], an operand of the
        sparse entry points.  A token that chose an expert twice would give two equal columns,
        which these do not take.  Reads the number of entries back."""
        n = int(self.pos[-1])
        order = self.order[:n].long()
        shape = torch.tensor([self.experts, self.tokens], dtype=torch.int32)
        return CSR_gpu(self.pos, (order // self.per_token).int(),
                       weights.detach().float().reshape(-1)[order], shape)


def gpu_route(experts: torch.Tensor, n_experts: int) -> Route:
    """Sort the choices `experts` (int32 or int64 [tokens, per_token]) by expert.  An id outside
    [0, n_experts) drops its entry.  At most 2048 experts."""
    device = _device_of(experts, "experts")
    if not 1 <= n_experts <= MAX_EXPERTS:
        raise ValueError(f"n_experts must be from 1 to {MAX_EXPERTS}, got {n_experts}")
    if experts.dim() == 2 and experts.shape[1] < 1:
        raise ValueError("experts: a token needs at least one choice")
    got = _call("route", device, experts, n_experts)
    if got is None:
        _check_tensor(experts, "experts", device, 2, (torch.int32, torch.int64))
        raise ValueError("gpu_route: refused operands")
    return Route(*got)


def _check_route(route):
    if not isinstance(route, Route):
        raise TypeError(f"route: expected a Route, got {type(route).__name__}")


def _refuse_rows(t, name, device, rows):
    _check_tensor(t, name, device, 2, _TYPES)
    if t.shape[0] != rows:
        raise ValueError(f"{name}: expected {rows} rows, got {t.shape[0]}")


def _dispatch(x, route):
    got = _call("dispatch", x.device, x, route.pos, route.slot)
    if got is None:
        _refuse_rows(x, "x", route.pos.device, route.tokens)
        raise ValueError("gpu_dispatch: refused operands")
    return got


def _combine(rows, weights, slot):
    got = _call("combine", rows.device, rows, weights, slot)
    if got is None:
        _refuse_rows(rows, "rows", slot.device, slot.numel())
        _check_tensor(weights, "weights", slot.device, 2, (torch.float32,))
        raise ValueError(f"weights: expected shape {tuple(slot.shape)}, got "
                         f"{tuple(weights.shape)}")
    return got


# The functions save the route's tensors, not the route, so that torch notices when one of them was
# written again before the backward pass.

def _saved(t):
    return t.clone() if t.is_inference() else t  # (torch saves none of inference mode)


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, route):
        ctx.save_for_backward(_saved(route.slot))
        return _dispatch(x, route)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, drows):
        slot, = ctx.saved_tensors
        return _combine(drows, None, slot), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, route):
        ctx.save_for_backward(rows, weights, _saved(route.pos), _saved(route.slot))
        return _combine(rows, weights, route.slot)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        rows, weights, pos, slot = ctx.saved_tensors
        drows, dweights = _call("combine_backward", rows.device, rows, weights, pos, slot, dout)
        return drows, dweights, None


def gpu_dispatch(x: torch.Tensor, route: Route) -> torch.Tensor:
    """Rows of x [tokens, width] by place, [tokens * per_token, width]: a token's row once for
    each of its experts, and zeros past the last expert's entries.  Differentiable in x."""
    _device_of(x, "x")
    _check_route(route)
    if _has_derivatives(x):
        return _Dispatch.apply(x, route)
    return _dispatch(x, route)


def gpu_combine(rows: torch.Tensor, route: Route, weights: torch.Tensor) -> torch.Tensor:
    """Each token's sum of its experts' rows times `weights` [tokens, per_token] (float32; other
    floating types are converted), [tokens, width] in the rows' type; dropped entries add
    nothing.  Differentiable in rows and weights."""
    _device_of(rows, "rows")
    _check_route(route)
    _device_of(weights, "weights")
    if weights.dtype != torch.float32 and weights.is_floating_point():
        weights = weights.float()
    if _has_derivatives(rows, weights):
        return _Combine.apply(rows, weights, route)
    return _combine(rows, weights, route.slot)
