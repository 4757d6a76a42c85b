"""Attention over blocks of keys that a score selects for each query.

A cache's keys are cut into blocks of 32, 64 or 128.  `gpu_block_means` summarises each block by
its mean key, `gpu_block_scores` scores the blocks for every query and key head,
`gpu_block_select` keeps the best of them, and `gpu_block_attention` attends to the keys of those
blocks alone; its gradients of q, k and v come through torch's autograd.

Layouts: q [batch, queries, q_heads, head_dim], k and v [batch, keys, kv_heads, head_dim], any
strides (a tensor whose rows are not whole 16-byte pieces apart is copied first), float32, float16
or bfloat16.  Head h of q uses key head h // (q_heads // kv_heads), and the heads of such a group
share the block ids.  `lengths` (int32 [batch], on the device) says how many keys each sequence
has; without it all `keys` rows count.  Query t stands at place lengths - queries + t of its
sequence: one new token of a cache is queries = 1, and a prompt is queries = keys.

Every call is asynchronous on torch's current stream, reads nothing back and may be captured in a
graph.  There is no CPU fallback.
"""

from __future__ import annotations

import functools
import math

import torch
from torch.autograd import forward_ad

from . import _device, _lib
from .ops import _entry

_TYPES = (torch.float32, torch.float16, torch.bfloat16)
_MOST_SCALE = torch.finfo(torch.float32).max


_BOUND: dict = {}


def _bind(name):
    fn = _BOUND[name] = functools.partial(getattr(_lib.load_bridge(), name),
                                          _entry("nacho_" + name))
    return fn


def _call(name, device, *args):
    """The bridge's call of entry point nacho_<name>; None for operands that it or the entry point
    refuses: the caller then names what is wrong."""
    fn = _BOUND.get(name) or _bind(name)
    index = device.index
    if torch._C._cuda_getDevice() == index:
        got = fn(torch._C._cuda_getCurrentRawStream(index), index, *args)
    else:
        with _device.on_device(device):
            got = fn(torch._C._cuda_getCurrentRawStream(index), index, *args)
    if type(got) is int:
        if got == -1:  # NACHO_ERR_INVALID_ARGUMENT
            return None
        _lib.check(got, "nacho_" + name)
    return got


def _device_of(t, name):
    if isinstance(t, torch.Tensor) and t.is_cuda:
        return t.device
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    raise ValueError(f"{name}: expected a GPU tensor, got device {t.device}")


# ---- what is wrong with refused operands ----------------------------------------------

def _check_tensor(t, name, device, dims, dtypes):
    if _device_of(t, name) != device:
        raise ValueError(f"operands on different devices: {device} and {t.device}")
    if t.dim() != dims:
        raise ValueError(f"{name}: expected {dims} dimensions, got shape {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: expected dtype {' or '.join(map(str, dtypes))}, got {t.dtype}")


def _check_lengths(lengths, device, batch):
    if lengths is not None:
        _check_tensor(lengths, "lengths", device, 1, (torch.int32,))
        if lengths.numel() != batch:
            raise ValueError(f"lengths: expected {batch} entries, got {lengths.numel()}")


def _check_heads(q_heads, kv_heads, head_dim, block):
    if kv_heads < 1 or q_heads < 1 or q_heads % kv_heads:
        raise ValueError(f"q has {q_heads} heads, not a multiple of the keys' {kv_heads}")
    if head_dim % 8 or not 8 <= head_dim <= 128:
        raise ValueError(f"head_dim must be a multiple of 8 from 8 to 128, got {head_dim}")
    _check_block(block)


def _check_block(block):
    if block not in (32, 64, 128):
        raise ValueError(f"block must be 32, 64 or 128, got {block}")


def _refuse_attention(q, k, v, blocks, lengths, block, scale):
    device = q.device
    _check_tensor(q, "q", device, 4, _TYPES)
    for t, name in ((k, "k"), (v, "v")):
        _check_tensor(t, name, device, 4, (q.dtype,))
    _check_heads(q.shape[2], k.shape[2], q.shape[3], block)
    if k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"shapes of q {tuple(q.shape)}, k {tuple(k.shape)} and v "
                         f"{tuple(v.shape)} do not fit")
    _check_tensor(blocks, "blocks", device, 4, (torch.int32,))
    want = (q.shape[0], q.shape[1], k.shape[2])
    if tuple(blocks.shape[:3]) != want:
        raise ValueError(f"blocks: expected shape {want} + (count,), got {tuple(blocks.shape)}")
    _check_lengths(lengths, device, q.shape[0])
    if abs(scale) > _MOST_SCALE / math.log2(math.e):  # (the exponentials are of base 2)
        raise ValueError(f"scale must be at most 2.3e38, got {scale}")
    raise ValueError("gpu_block_attention: refused operands (more than 2^31 - 1 rows, or more "
                     "than 1024 heads of q to a key head)")


def _scale(scale, shape):
    if scale is None:
        return (shape[-1] or 1) ** -0.5 if shape else 1.0
    if not abs(scale) <= _MOST_SCALE:  # (NaN too)
        raise ValueError(f"scale must be finite in float32, got {scale}")
    return float(scale)


# ---- means, scores, selection ---------------------------------------------------------

def gpu_block_means(k: torch.Tensor, block: int,
                    lengths: torch.Tensor | None = None) -> torch.Tensor:
    """Mean key of each block, float32 [batch, ceil(keys / block), kv_heads, head_dim], over the
    keys within the sequence's length; 0 for a block without any.  No gradient."""
    device = _device_of(k, "k")
    got = _call("block_means", device, k, lengths, block)
    if got is None:
        _check_tensor(k, "k", device, 4, _TYPES)
        _check_heads(1, 1, k.shape[3], block)
        _check_lengths(lengths, device, k.shape[0])
        raise ValueError("gpu_block_means: refused operands")
    return got


def gpu_block_scores(q: torch.Tensor, means: torch.Tensor, block: int, keys: int,
                     lengths: torch.Tensor | None = None, causal: bool = True,
                     scale: float | None = None) -> torch.Tensor:
    """Score of every block for every query and key head, float32 [batch, queries, kv_heads,
    blocks]: scale (1 / sqrt(head_dim) unless given) times the sum of the group's heads of q,
    times the block's mean key (`means`, as gpu_block_means gives it).  -inf for a block that
    starts after the query's place, or not causal, at the sequence's end.  `keys`: rows of the
    cache.  No gradient."""
    device = _device_of(q, "q")
    got = _call("block_scores", device, q, means, lengths, block, keys, bool(causal),
                _scale(scale, q.shape))
    if got is not None:
        return got
    _check_tensor(q, "q", device, 4, _TYPES)
    _check_tensor(means, "means", device, 4, (torch.float32,))
    _check_heads(q.shape[2], means.shape[2], q.shape[3], block)
    _check_lengths(lengths, device, q.shape[0])
    raise ValueError(f"means: expected [{q.shape[0]}, ceil({keys} / {block}), kv_heads, "
                     f"{q.shape[3]}], got {tuple(means.shape)}")


def gpu_block_select(scores: torch.Tensor, count: int, block: int, keys: int,
                     lengths: torch.Tensor | None = None, causal: bool = True, sink: int = 1,
                     local: int = 1) -> torch.Tensor:
    """Block ids of every query and key head, int32 [batch, queries, kv_heads, count], ascending
    and -1 behind: the `local` latest blocks up to the query's own and the first `sink` blocks,
    whatever their scores, then those of the highest scores, equal ones lowest id first.  A block
    with a score of -inf or NaN is taken only as one of the former."""
    device = _device_of(scores, "scores")
    if count < 0 or not 0 <= sink <= 1 << 20 or not 0 <= local <= 1 << 20:
        raise ValueError(f"count, sink and local must be >= 0 (sink and local <= 2^20), got "
                         f"{count}, {sink} and {local}")
    got = _call("block_select", device, scores, lengths, count, block, keys, bool(causal), sink,
                local)
    if got is None:
        _check_tensor(scores, "scores", device, 4, (torch.float32,))
        _check_block(block)
        _check_lengths(lengths, device, scores.shape[0])
        raise ValueError(f"scores: expected ceil({keys} / {block}) blocks, got "
                         f"{tuple(scores.shape)}")
    return got


# ---- attention ------------------------------------------------------------------------

def _has_derivatives(*tensors):
    """Whether autograd is to know of a call with these operands.  (A tangent does not show in
    requires_grad, and the autograd functions, which have none, refuse it.)"""
    if torch.is_grad_enabled():
        for t in tensors:
            if getattr(t, "requires_grad", False):
                return True
    return forward_ad._current_level >= 0


class _BlockAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, blocks, lengths, block, causal, scale):
        got = _call("block_attention", q.device, q, k, v, blocks, lengths, block, causal, scale,
                    True)
        if got is None:
            _refuse_attention(q, k, v, blocks, lengths, block, scale)
        out, lse = got
        ctx.save_for_backward(q, k, v, blocks, lengths, out, lse)
        ctx.how = block, causal, scale
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)  # (lse's would be a launch that fills zeros)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        q, k, v, blocks, lengths, out, lse = ctx.saved_tensors
        grads = None, None, None
        if dout is not None:
            grads = _call("block_attention_backward", q.device, q, k, v, blocks, lengths, *ctx.how,
                          dout, out, lse)
        return (*grads, None, None, None, None, None)


def gpu_block_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, blocks: torch.Tensor,
                        block: int, lengths: torch.Tensor | None = None, causal: bool = True,
                        scale: float | None = None, return_lse: bool = False):
    """softmax(scale q k^T) v over the keys of each query's blocks, [batch, queries, q_heads,
    head_dim] in q's type (scale: 1 / sqrt(head_dim) unless given).

    `blocks`: int32 [batch, queries, kv_heads, count] ids in any order; an id outside the sequence
    is no block and a repeated one counts once.  Causal: only keys up to the query's place.  A
    query that sees nothing gives 0.  With `return_lse` also the log of the sum of exponentials,
    float32 [batch, queries, q_heads] (-inf for such a query; no gradient), with which results
    over disjoint sets of keys can be joined.  Differentiable in q, k and v (in backward mode,
    once)."""
    device = _device_of(q, "q")
    scale = _scale(scale, q.shape)
    causal = bool(causal)
    if _has_derivatives(q, k, v):
        out, lse = _BlockAttention.apply(q, k, v, blocks, lengths, block, causal, scale)
        return (out, lse) if return_lse else out
    got = _call("block_attention", device, q, k, v, blocks, lengths, block, causal, scale,
                return_lse)
    if got is None:
        _refuse_attention(q, k, v, blocks, lengths, block, scale)
    return got if return_lse else got[0]


def gpu_block_attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                                 v: torch.Tensor, blocks: torch.Tensor, block: int,
                                 out: torch.Tensor, lse: torch.Tensor,
                                 lengths: torch.Tensor | None = None, causal: bool = True,
                                 scale: float | None = None):
    """(dq, dk, dv) of gpu_block_attention from its output's gradient, its operands and its
    results, for callers that keep their own record of a step.  Deterministic."""
    device = _device_of(q, "q")
    scale = _scale(scale, q.shape)
    got = _call("block_attention_backward", device, q, k, v, blocks, lengths, block, bool(causal),
                scale, dout, out, lse)
    if got is None:
        for t, name in ((dout, "dout"), (out, "out")):
            _check_tensor(t, name, device, 4, (q.dtype,))
            if t.shape != q.shape:
                raise ValueError(f"{name}: expected shape {tuple(q.shape)}, got {tuple(t.shape)}")
        _check_tensor(lse, "lse", device, 3, (torch.float32,))
        if lse.shape != q.shape[:3]:
            raise ValueError(f"lse: expected shape {tuple(q.shape[:3])}, got {tuple(lse.shape)}")
        _refuse_attention(q, k, v, blocks, lengths, block, scale)
    return got
