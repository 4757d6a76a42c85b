"""Block attention of 16-bit rows, where a sequence has few of them, and its gradients are as exact
as the formulas in float32 with the result rounded once.

The share that is allowed: a probability (or a score's gradient) reaches its product within 2^-15
(bfloat16) or 2^-20 (float16) of itself, its float32 exponential within about 2^-19; the result's
rounding is 2^-9 and 2^-12 of it on average.  These errors are independent, so they add in squares:
at most a hundredth of the last one's square is another 0.5%.  1.02 leaves room for that and for
the sample's own spread."""

import pytest
import torch

import nacho_amd
from tests import block_exact as exact
from tests import block_reference as ref
from tests.test_gpu_blocks import FEW, MANY, WIDE, _operands

pytestmark = pytest.mark.gpu

TYPES = (torch.float16, torch.bfloat16)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes", [FEW[2], FEW[4], FEW[7], (64, 1, 300, 32, 8, 128, 64, 3),
                                   (64, 1, 290, 32, 8, 64, 32, 3), (130, 3, 90, 14, 2, 80, 128, 1),
                                   (128, 1, 70, 16, 8, 96, 32, 2)],
                         ids=str)
def test_output_is_rounded_once(gpu, sizes, dtype):
    q, k, v, ids, _ = _operands(41, dtype, *sizes)
    see = ref.visible(ids, sizes[1], sizes[2], sizes[6], None, True)
    want = exact.attention(q, k, v, see)
    got = nacho_amd.gpu_block_attention(q.to(gpu), k.to(gpu), v.to(gpu), ids.to(gpu), sizes[6])
    exact.rounded_once(got, want, "out")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_infinite_values_stay_infinities(gpu, dtype):
    """A value that is infinite is a query's result in that column, where the query sees it."""
    for sizes in (FEW[3], FEW[8], MANY[2], WIDE[0]):
        q, k, v, ids, _ = _operands(42, dtype, *sizes)
        v[:, 5, :, 2], v[:, 37, :, 3] = float("inf"), float("-inf")
        see = ref.visible(ids, sizes[1], sizes[2], sizes[6], None, True)
        group = sizes[3] // sizes[4]
        got = nacho_amd.gpu_block_attention(q.to(gpu), k.to(gpu), v.to(gpu), ids.to(gpu),
                                            sizes[6]).cpu()
        for key, col, value in ((5, 2, float("inf")), (37, 3, float("-inf"))):
            sees = see[..., key].transpose(1, 2).repeat_interleave(group, -1)
            assert (got[..., col][sees] == value).all()
            assert torch.isfinite(got[..., col][~sees]).all()


def _gradients(gpu, q, k, v, ids, dout, block):
    """The gradients, and what they are by their formulas (delta of the output that was given)."""
    dev = [x.to(gpu).requires_grad_() for x in (q, k, v)]
    out = nacho_amd.gpu_block_attention(*dev, ids.to(gpu), block)
    grads = torch.autograd.grad(out, dev, dout.to(gpu))
    see = ref.visible(ids, q.shape[1], k.shape[1], block, None, True)
    return grads, exact.attention(q, k, v, see, out.detach().cpu(), dout)[1:]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes", [FEW[6], FEW[7], *MANY[:3], WIDE[1]], ids=str)
def test_gradients_are_rounded_once(gpu, sizes, dtype):
    got, want = _gradients(gpu, *_operands(43, dtype, *sizes), sizes[6])
    for x, y, name in zip(got, want, ("dq", "dk", "dv")):
        exact.rounded_once(x, y, name)


@pytest.mark.parametrize("size", (1e-4, 8e3))
@pytest.mark.parametrize("sizes", [(1, 65, 130, 6, 2, 128, 64, 2), (2, 90, 333, 4, 4, 64, 32, 5),
                                   MANY[0]], ids=str)
def test_float16_gradients_of_small_and_large_steps(gpu, sizes, size):
    """Gradients of a scaled loss: where float16 holds the results, it does not matter that it
    would not hold the scores' gradients."""
    q, k, v, ids, dout = _operands(44, torch.float32, *sizes)
    q, k = 0.3 * q, 0.3 * k
    dout = (dout * size).clamp(-60000, 60000)
    operands = [x.half() if x.is_floating_point() else x for x in (q, k, v, ids, dout)]
    got, want = _gradients(gpu, *operands, sizes[6])
    for x, y, name in zip(got, want, ("dq", "dk", "dv")):
        assert y.abs().max() < 65000, name
        exact.rounded_once(x, y, name)


def test_float16_gradients_of_small_probabilities(gpu):
    """Queries that see thousands of keys: probabilities down to 2^-20 and below."""
    q, k, v, _, dout = _operands(45, torch.float16, 1, 40, 4096, 4, 2, 64, 128, 1)
    ids = torch.arange(32, dtype=torch.int32).expand(1, 40, 2, 32).contiguous()
    got, want = _gradients(gpu, 1.5 * q, k, v, ids, dout, 128)
    for x, y, name in zip(got, want, ("dq", "dk", "dv")):
        exact.rounded_once(x, y, name)


SMALL, LARGE = (1e-4, 1.0), (8e3, 8.0)  # of dout and of v


@pytest.mark.parametrize("sizes", [(1, 65, 130, 6, 2, 128, 64, 2), (2, 90, 333, 4, 4, 64, 32, 5),
                                   (1, 70, 140, 3, 3, 72, 128, 1)], ids=str)
@pytest.mark.parametrize("size", (SMALL, LARGE), ids=str)
def test_float16_gradients_of_small_and_large_steps(gpu, sizes, size):
    """Gradients of a scaled loss: where float16 holds the results, it does not matter that it
    would not hold the scores' gradients."""
    q, k, v, ids, dout = _operands(44, torch.float32, *sizes)
    q, k, v = 0.3 * q, 0.3 * k, size[1] * v
    dout = (dout * size[0]).clamp(-60000, 60000)
    operands = [x.half() if x.is_floating_point() else x for x in (q, k, v, ids, dout)]
    got, want = _gradients(gpu, *operands, sizes[6])
    for x, y, name in zip(got, want, ("dq", "dk", "dv")):
        assert y.abs().max() < 65000, name
        exact.rounded_once(x, y, name)


def test_float16_gradients_of_small_probabilities(gpu):
    """Queries that see thousands of keys: probabilities down to 2^-20 and below."""
    q, k, v, _, dout = _operands(45, torch.float16, 1, 40, 4096, 4, 2, 64, 128, 1)
    ids = torch.arange(32, dtype=torch.int32).expand(1, 40, 2, 32).contiguous()
    got, want = _gradients(gpu, 1.5 * q, k, v, ids, dout, 128)
    for x, y, name in zip(got, want, ("dq", "dk", "dv")):
        exact.rounded_once(x, y, name)
