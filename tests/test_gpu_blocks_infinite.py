"""Keys and values that are not finite in places that a query sees, or that nobody sees: results are
those of the formulas, and no finite number stands where these have none."""

import math

import pytest
import torch

import nacho_amd
from tests import block_exact as exact
from tests import block_reference as ref
from tests.test_gpu_blocks import FEW, MANY, TYPES, WIDE, _operands

pytestmark = pytest.mark.gpu

# what a finite result may be off, in parts of what rounding it is: these tests look for other values
NEAR = {torch.float32: 200.0, torch.float16: 2.0, torch.bfloat16: 2.0}


def _sees(ids, sizes, key):
    see = ref.visible(ids, sizes[1], sizes[2], sizes[6], None, True)
    return see, see[..., key].transpose(1, 2).repeat_interleave(sizes[3] // sizes[4], -1)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes", [FEW[3], FEW[8], MANY[0], WIDE[0]], ids=str)
def test_keys_whose_score_is_minus_infinity(gpu, sizes, dtype):
    """Such a key has probability 0: it is as good as unseen, but dq is 0 times infinity in the
    column that holds the infinity."""
    q, k, v, ids, dout = _operands(51, dtype, *sizes)
    key, col = 3, 1
    q[..., col] = q[..., col].abs() + 0.25
    k[:, key, :, col] = -math.inf
    see, sees = _sees(ids, sizes, key)
    dev = [x.to(gpu).requires_grad_() for x in (q, k, v)]
    out = nacho_amd.gpu_block_attention(*dev, ids.to(gpu), sizes[6])
    grads = [x.cpu() for x in torch.autograd.grad(out, dev, dout.to(gpu))]
    see = see.clone()
    see[..., key] = False
    k[:, key, :, col] = 0.0
    want = exact.attention(q, k, v, see, out.detach().cpu(), dout)
    exact.rounded_once(out, want[0], "out", NEAR[dtype])
    assert sees.any()
    assert torch.isnan(grads[0][..., col][sees]).all()
    grads[0][..., col] = torch.where(sees, 0.0, grads[0][..., col])
    want[1][..., col] = torch.where(sees, 0.0, want[1][..., col])
    for x, y, name in zip(grads, want[1:], ("dq", "dk", "dv")):
        exact.rounded_once(x, y, name, NEAR[dtype])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes", [(2, 1, 200, 4, 2, 72, 64, 4), FEW[3], FEW[8], MANY[0], WIDE[0]],
                         ids=str)
def test_infinite_values_of_the_least_probabilities(gpu, sizes, dtype):
    """An infinity times a probability that is too small for its type is not left out."""
    q, k, v, ids, _ = _operands(52, dtype, *sizes)
    key, col = 3, 1
    q[..., 0] = q[..., 0].abs() + 1.0
    k[:, key] = 0.0
    k[:, key, :, 0] = -2000.0  # a score of less than -150
    v[:, key, :, col] = math.inf
    see, sees = _sees(ids, sizes, key)
    got = nacho_amd.gpu_block_attention(q.to(gpu), k.to(gpu), v.to(gpu), ids.to(gpu),
                                        sizes[6]).cpu()
    first = torch.zeros(sizes[2], dtype=torch.bool)
    first[key] = True
    alone = (see & ~first).any(-1).transpose(1, 2).repeat_interleave(sizes[3] // sizes[4], -1)
    assert (sees & alone).any()
    assert not torch.isfinite(got[..., col][sees & alone]).any()
    v[:, key, :, col] = 0.0
    want = exact.attention(q, k, v, see)
    got[..., col] = torch.where(sees, 0.0, got[..., col])
    want[..., col] = torch.where(sees, 0.0, want[..., col])
    exact.rounded_once(got, want, "out", NEAR[dtype])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("block", (32, 64, 128))
@pytest.mark.parametrize("dim", (64, 128))
def test_gradients_of_keys_that_nobody_sees(gpu, dim, block, dtype):
    """One query sees an infinite value: its block's later keys and values, infinite ones among
    them, which it does not see, keep a gradient of 0."""
    q, k, v, ids, dout = _operands(53, dtype, 1, block, block, 2, 1, dim, block, 1)
    ids[:] = -1
    ids[:, 10] = 0
    v[:, 3], v[:, 20], k[:, 21] = math.inf, -math.inf, math.nan
    dev = [x.to(gpu).requires_grad_() for x in (q, k, v)]
    out = nacho_amd.gpu_block_attention(*dev, ids.to(gpu), block)
    _, dk, dv = torch.autograd.grad(out, dev, dout.to(gpu))
    assert not torch.isfinite(dk[:, :11]).any()
    assert not dk[:, 11:].any() and not dv[:, 11:].any()


@pytest.mark.parametrize("scale", (2.4e38, -3e38, 1e39, math.nan))
def test_scales_past_the_range_are_named(gpu, scale):
    q, k, v, ids, dout = (x.to(gpu) for x in _operands(54, torch.float32, *FEW[3]))
    f = nacho_amd.gpu_block_attention
    out, lse = f(q, k, v, ids, 64, return_lse=True)
    with pytest.raises(ValueError, match="scale must be"):
        f(q, k, v, ids, 64, scale=scale)
    with pytest.raises(ValueError, match="scale must be"):
        f(q.clone().requires_grad_(), k, v, ids, 64, scale=scale)
    with pytest.raises(ValueError, match="scale must be"):
        nacho_amd.gpu_block_attention_backward(dout, q, k, v, ids, 64, out, lse, scale=scale)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim,block", [(64, 64), (128, 64), (96, 32)])
def test_infinite_score_gradients(gpu, dim, block, dtype):
    """A query that sees an infinite value takes its infinity from the other keys' score gradients:
    their dk is that infinity with the query's signs."""
    q, k, v, _, dout = _operands(55, dtype, 1, 1, 40, 1, 1, dim, block, 1)
    ids = torch.arange((40 + block - 1) // block, dtype=torch.int32).view(1, 1, 1, -1)
    dout[..., 0], v[:, 7, :, 0] = 1.0, math.inf
    q = torch.where(q.abs() < 0.25, 0.25, q)
    dev = [x.to(gpu).requires_grad_() for x in (q, k, v)]
    out = nacho_amd.gpu_block_attention(*dev, ids.to(gpu), block)
    dq, dk, dv = (x.cpu() for x in torch.autograd.grad(out, dev, dout.to(gpu)))
    assert torch.isnan(dq).all() and torch.isnan(dk[:, 7]).all() and torch.isfinite(dv).all()
    others = torch.arange(40) != 7
    assert torch.equal(dk[:, others].float(), (-math.inf * q.sign().float()).expand(1, 39, 1, dim))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes", [(2, 1, 200, 4, 2, 72, 64, 4), (1, 3, 200, 4, 2, 128, 32, 7),
                                   (64, 1, 200, 32, 8, 64, 64, 4)], ids=str)
@pytest.mark.parametrize("behind", (8.0, 10.0, 12.0, 14.0, 16.0))
def test_infinite_values_of_small_probabilities(gpu, sizes, behind, dtype):
    """A value that is infinite makes the result that infinity, whatever share its key has, down to
    the least probability that the type holds (2^-24 of the largest in float16)."""
    batch, queries, keys, heads, kv_heads, dim, block, count = sizes
    g = torch.Generator().manual_seed(56)
    q = torch.zeros(batch, queries, heads, dim, dtype=dtype)
    k = torch.zeros(batch, keys, kv_heads, dim, dtype=dtype)
    v = torch.randn(batch, keys, kv_heads, dim, generator=g).to(dtype)
    q[..., 0] = 1.0
    k[:, 3, :, 0], k[:, 70, :, 0] = -behind, -behind - 0.375
    v[:, 3, :, 1], v[:, 70, :, 2] = math.inf, -math.inf
    ids = torch.arange(count, dtype=torch.int32).expand(batch, queries, kv_heads, count)
    got = nacho_amd.gpu_block_attention(*(x.to(gpu) for x in (q, k, v, ids.contiguous())), block,
                                        scale=1.0).cpu()
    assert (got[..., 1] == math.inf).all() and (got[..., 2] == -math.inf).all()
    assert torch.isfinite(got[..., 3:]).all()
