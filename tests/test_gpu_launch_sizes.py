"""Operators on more rows than a launch has workgroups for: 2^24 workgroups of 256 threads are 2^32
work-items, of which a launch would run none."""

import pytest
import torch

import nacho_amd

pytestmark = pytest.mark.gpu

TOKENS = (1 << 26) + 8  # four wavefronts of a workgroup have one each


def test_routing(gpu):
    choices = torch.ones(TOKENS, 1, dtype=torch.int32, device=gpu)
    choices[::3] = 0
    choices[5::1001] = -1
    route = nacho_amd.gpu_route(choices, 2)
    x = torch.arange(TOKENS, device=gpu, dtype=torch.int32).remainder_(251).bfloat16()
    x = x[:, None].repeat(1, 2).requires_grad_()
    rows = nacho_amd.gpu_dispatch(x, route)
    held = int(route.pos[2])
    assert torch.equal(rows.detach()[:held], x.detach()[route.order[:held].long()])
    assert not rows.detach()[held:].any()
    w = torch.full((TOKENS, 1), 0.5, device=gpu).requires_grad_()
    there = (choices >= 0).expand_as(x)
    out = nacho_amd.gpu_combine(rows, route, w)
    assert torch.equal(out, torch.where(there, 0.5 * x, 0.0))
    dx, dw = torch.autograd.grad(out, (x, w), torch.ones_like(out))
    assert torch.equal(dx, torch.where(there, 0.5, 0.0).bfloat16())
    assert torch.equal(dw, torch.where(there[:, :1], 2 * x[:, :1].float(), 0.0))


def test_select(gpu):
    got = nacho_amd.gpu_block_select(torch.zeros(1, TOKENS, 1, 1, device=gpu), 1, 32, 32)
    want = torch.full((1, TOKENS, 1, 1), -1, dtype=torch.int32, device=gpu)
    want[0, -32:] = 0  # the queries that stand in the sequence
    assert torch.equal(got, want)


def test_means(gpu):
    k = torch.ones(1, 32, 1, 8, device=gpu).expand((1 << 24) + 3, 32, 1, 8)
    assert torch.equal(nacho_amd.gpu_block_means(k, 32).sum(), torch.tensor(8.0 * len(k)).to(gpu))
