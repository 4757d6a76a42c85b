"""The two ends of a language model's step: words to rows, and rows to a loss over the words.

`gpu_embedding` looks rows up in a table, scaled, and its gradient sums the tokens of each word,
sorted by word.  `gpu_linear_cross_entropy` is the cross entropy of rows times a table (often the
same one) against target words, with its gradients, and never has the logits in memory: it goes
over the vocabulary in pieces, and over the tokens that have a target alone.

Rows and tables are float32, float16 or bfloat16, those of a call alike; ids are int32 or int64, and
an id that is no word is none: its row is zeros, its loss 0, and it has no part in any gradient.
Sums are float32 and have a fixed order.

Calls are asynchronous on torch's current stream, read nothing back and may be captured in a
graph.  There is no CPU fallback.
"""

from __future__ import annotations

import torch

from .blocks import _MOST_SCALE, _TYPES, _call, _check_tensor, _device_of, _has_derivatives
from .routing import _saved

MAX_WORDS = 1 << 30

_IDS = (torch.int32, torch.int64)
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}  # NACHO_LOSS_NONE ...


def _factor(scale):
    if not abs(scale) <= _MOST_SCALE:  # (NaN too)
        raise ValueError(f"scale must be finite in float32, got {scale}")
    return float(scale)


def _check_any(t, name, device, dtypes):
    if _device_of(t, name) != device:
        raise ValueError(f"operands on different devices: {device} and {t.device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: expected dtype {' or '.join(map(str, dtypes))}, got {t.dtype}")


def _check_words(words):
    if not 0 <= words <= MAX_WORDS:
        raise ValueError(f"words must be from 0 to {MAX_WORDS}, got {words}")


def _check_shape(t, name, shape):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")


# ---- embedding ------------------------------------------------------------------------

def _embedding(table, ids, scale):
    got = _call("embedding", table.device, ids, table, scale)
    if got is None:
        _check_tensor(table, "table", table.device, 2, _TYPES)
        _check_any(ids, "ids", table.device, _IDS)
        _check_words(table.shape[0])
        raise ValueError("gpu_embedding: refused operands")
    return got


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale):
        out = _embedding(table, ids, scale)
        ctx.save_for_backward(_saved(ids))
        ctx.how = table.shape[0], scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        ids, = ctx.saved_tensors
        return _call("embedding_backward", dout.device, dout, ids, *ctx.how), None, None


def gpu_embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """Rows of table [words, width] by id, times scale: ids' shape + [width], in the table's type;
    zeros for an id outside [0, words).  Differentiable in table (in backward mode, once)."""
    _device_of(ids, "ids")
    _device_of(table, "table")
    scale = _factor(scale)
    if _has_derivatives(table):
        return _Embedding.apply(table, ids, scale)
    return _embedding(table, ids, scale)


def gpu_embedding_backward(dout: torch.Tensor, ids: torch.Tensor, words: int,
                           scale: float = 1.0) -> torch.Tensor:
    """The gradient of gpu_embedding's table, [words, width], from that of its result: a word's
    row is scale times the sum of its tokens' rows of dout, in a fixed order."""
    device = _device_of(dout, "dout")
    scale = _factor(scale)
    _check_words(words)
    got = _call("embedding_backward", device, dout, ids, words, scale)
    if got is None:
        _check_any(ids, "ids", device, _IDS)
        _check_any(dout, "dout", device, _TYPES)
        if dout.dim() != ids.dim() + 1 or dout.shape[:-1] != ids.shape:
            raise ValueError(f"dout: expected shape {tuple(ids.shape)} + (width,), got "
                             f"{tuple(dout.shape)}")
        raise ValueError("gpu_embedding_backward: refused operands")
    return got


# ---- linear cross entropy ---------------------------------------------------------------

def _refuse_loss(x, table, targets):
    device = x.device
    _check_any(x, "x", device, _TYPES)
    _check_tensor(table, "table", device, 2, (x.dtype,))
    _check_any(targets, "targets", device, _IDS)
    if x.dim() < 1 or x.shape[-1] != table.shape[1]:
        raise ValueError(f"x: expected rows of {table.shape[1]}, got shape {tuple(x.shape)}")
    _check_shape(targets, "targets", x.shape[:-1])
    if min(table.shape) < 1:
        raise ValueError(f"table: expected words and columns, got shape {tuple(table.shape)}")
    raise ValueError("gpu_linear_cross_entropy: refused operands (more than 2^30 words or tokens, "
                     "or more than 2^20 columns)")


def _reduction(name):
    if name not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'mean' or 'sum', got {name!r}")
    return _REDUCTIONS[name]


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, table, targets, scale, reduction):
        got = _call("linear_cross_entropy", x.device, x, table, targets, scale, reduction, True)
        if got is None:
            _refuse_loss(x, table, targets)
        loss, stats = got
        ctx.save_for_backward(x, table, _saved(targets), stats)
        ctx.how = scale, reduction
        ctx.mark_non_differentiable(stats)
        ctx.set_materialize_grads(False)
        return loss, stats

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss, _):
        dx = dtable = None
        if dloss is not None:
            x, table, targets, stats = ctx.saved_tensors
            dx, dtable = _call("linear_cross_entropy_backward", x.device, x, table, targets,
                               stats, dloss, *ctx.how, *ctx.needs_input_grad[:2])
        return dx, dtable, None, None, None


def gpu_linear_cross_entropy(x: torch.Tensor, table: torch.Tensor, targets: torch.Tensor,
                             scale: float = 1.0, reduction: str = "mean",
                             return_stats: bool = False):
    """Cross entropy of scale x table^T against targets, without the logits in memory: for rows x
    [..., width], table [words, width] and targets [...], log(sum_w exp(z_w)) - z_target, float32.

    A target outside [0, words) leaves its token out: its loss is 0, it has no part in a gradient
    whatever its row holds, and does not count in a mean (of no token: 0).  reduction: 'none' (a
    loss per token), 'mean' or 'sum'.  With `return_stats` also what the backward pass needs,
    float32 [2, tokens]: each token's greatest logit and the sum of exp(logit - greatest), for the
    log of the sum of exponentials among others (0 and 1 where there is no target; no gradient).
    Differentiable in x and table (in backward mode, once)."""
    device = _device_of(x, "x")
    scale = _factor(scale)
    how = _reduction(reduction)
    if _has_derivatives(x, table):
        got = _LinearCrossEntropy.apply(x, table, targets, scale, how)
    else:
        got = _call("linear_cross_entropy", device, x, table, targets, scale, how,
                    bool(return_stats))
        if got is None:
            _refuse_loss(x, table, targets)
    return tuple(got) if return_stats else got[0]


def gpu_linear_cross_entropy_backward(dloss: torch.Tensor, x: torch.Tensor, table: torch.Tensor,
                                      targets: torch.Tensor, stats: torch.Tensor,
                                      scale: float = 1.0, reduction: str = "mean"):
    """(dx, dtable) of gpu_linear_cross_entropy from its result's gradient (float32), its operands
    and its stats, for callers that keep their own record of a step.  Deterministic."""
    device = _device_of(x, "x")
    scale = _factor(scale)
    how = _reduction(reduction)
    got = _call("linear_cross_entropy_backward", device, x, table, targets, stats, dloss, scale,
                how, True, True)
    if got is None:
        _check_any(dloss, "dloss", device, (torch.float32,))
        _check_tensor(stats, "stats", device, 2, (torch.float32,))
        _check_any(targets, "targets", device, _IDS)
        _check_shape(stats, "stats", (2, targets.numel()))
        _check_shape(dloss, "dloss", targets.shape if reduction == "none" else ())
        _refuse_loss(x, table, targets)
    return got
