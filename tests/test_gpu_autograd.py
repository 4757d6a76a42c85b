"""What the differentiable operators do with other uses of torch's autograd: forward-mode
derivatives, which they do not have, are refused, and operands that are written again between the
passes are noticed."""

import pytest
import torch
from torch.autograd import forward_ad

import nacho_amd

pytestmark = pytest.mark.gpu


def _attention(gpu):
    q = torch.randn(1, 3, 4, 32, device=gpu)
    k, v = torch.randn(2, 1, 40, 2, 32, device=gpu)
    return [q, k, v], torch.zeros(1, 3, 2, 1, dtype=torch.int32, device=gpu)


@pytest.mark.parametrize("which", range(3))
def test_attention_refuses_tangents(gpu, which):
    ops, ids = _attention(gpu)
    with forward_ad.dual_level():
        nacho_amd.gpu_block_attention(*ops, ids, 32)  # (without one all is as it was)
        ops[which] = forward_ad.make_dual(ops[which], torch.ones_like(ops[which]))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="jvp"):
                nacho_amd.gpu_block_attention(*ops, ids, 32)


def test_routing_refuses_tangents(gpu):
    route = nacho_amd.gpu_route(torch.tensor([[0, 1], [1, 2]], device=gpu), 3)
    x, rows, w = (torch.randn(*s, device=gpu) for s in ((2, 8), (4, 8), (2, 2)))
    with forward_ad.dual_level():
        dual = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, rows, w)]
        with pytest.raises(NotImplementedError, match="jvp"):
            nacho_amd.gpu_dispatch(dual[0], route)
        for args in ((dual[1], route, w), (rows, route, dual[2]),
                     (rows, route, forward_ad.make_dual(w.half(), torch.ones_like(w).half()))):
            with pytest.raises(NotImplementedError, match="jvp"):
                nacho_amd.gpu_combine(*args)


@pytest.mark.parametrize("written", ("pos", "slot"))
def test_a_route_that_is_written_again_is_noticed(gpu, written):
    route = nacho_amd.gpu_route(torch.tensor([[0, 1], [1, 2]], device=gpu), 3)
    x, rows, w = (torch.randn(*s, device=gpu).requires_grad_() for s in ((2, 8), (4, 8), (2, 2)))
    there = nacho_amd.gpu_dispatch(x, route), nacho_amd.gpu_combine(rows, route, w)
    getattr(route, written).copy_(getattr(route, written).clone())
    if written == "slot":
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            there[0].sum().backward()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        there[1].sum().backward()


def test_a_route_of_inference_mode(gpu):
    choices = torch.tensor([[0, 1], [1, 2]], device=gpu)
    with torch.inference_mode():
        route = nacho_amd.gpu_route(choices, 3)
    x, rows, w = (torch.randn(*s, device=gpu).requires_grad_() for s in ((2, 8), (4, 8), (2, 2)))
    outs = [nacho_amd.gpu_dispatch(x, route), nacho_amd.gpu_combine(rows, route, w)]
    got = torch.autograd.grad(outs, (x, rows, w), [torch.ones_like(o) for o in outs])
    route = nacho_amd.gpu_route(choices, 3)
    outs = [nacho_amd.gpu_dispatch(x, route), nacho_amd.gpu_combine(rows, route, w)]
    want = torch.autograd.grad(outs, (x, rows, w), [torch.ones_like(o) for o in outs])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
