"""A training step's ends on more tokens than a launch has workgroups for, and on tables of more elements
than 32 bits count."""

import pytest
import torch

import nacho_amd
from tests.loss_reference import Loss, near

pytestmark = pytest.mark.gpu


def test_embedding_of_many_tokens(gpu):
    tokens = (1 << 26) + 8  # four wavefronts of a workgroup have one each
    ids = torch.arange(tokens, device=gpu, dtype=torch.int32).remainder_(300)
    ids[5::1001] = -1
    table = torch.arange(600, device=gpu, dtype=torch.float32).view(300, 2)
    rows = nacho_amd.gpu_embedding(ids, table)
    there = (ids >= 0)[:, None]
    assert torch.equal(rows, torch.where(there, table[ids.clamp(min=0).long()], 0.0))
    dtable = nacho_amd.gpu_embedding_backward(torch.ones_like(rows), ids, 300)
    count = torch.bincount(ids.clamp(min=0)[ids >= 0], minlength=300).float()
    assert torch.equal(dtable, count[:, None].expand(300, 2))  # (whole numbers of less than 2^24)


def test_embedding_of_a_large_table(gpu):
    words, width = 36_000_000, 64  # more elements than 32 bits count
    table = torch.zeros(words, width, dtype=torch.bfloat16, device=gpu)
    some = torch.tensor([0, 1, words // 2, words - 2, words - 1], device=gpu)
    table[some] = torch.arange(5, device=gpu)[:, None].bfloat16() + 1
    rows = nacho_amd.gpu_embedding(some, table)
    assert torch.equal(rows[:, 0].float(), torch.arange(5, device=gpu).float() + 1)
    del table
    dtable = nacho_amd.gpu_embedding_backward(rows, some, words)
    assert torch.equal(dtable[some], rows)
    assert float(dtable.sum(dtype=torch.float32)) == 64 * 15.0


def test_loss_of_many_tokens(gpu):
    tokens, words, width = 1_000_003, 40, 16
    g = torch.Generator(device=gpu).manual_seed(1)
    x = torch.randn(tokens, width, generator=g, device=gpu).bfloat16()
    table = torch.randn(words, width, generator=g, device=gpu).bfloat16()
    targets = torch.randint(-1, words, (tokens,), generator=g, device=gpu)
    xd, td = x.requires_grad_(), table.requires_grad_()
    loss = nacho_amd.gpu_linear_cross_entropy(xd, td, targets, reduction="sum")
    dloss = torch.tensor(1e-3, device=gpu)
    want = Loss(x, table, targets, reduction="sum", dloss=dloss)
    near(loss, want.loss, want.loss_off, "loss")
    dx, dtable = torch.autograd.grad(loss, (xd, td), dloss)
    near(dx, want.dx, want.dx_off, "dx")
    near(dtable, want.dtable, want.dtable_off, "dtable")


def test_loss_of_a_large_table(gpu):
    words, width = 270_000, 8192  # more elements than 32 bits count
    g = torch.Generator(device=gpu).manual_seed(2)
    table = torch.randn(words, width, generator=g, device=gpu).mul_(0.01).bfloat16()
    targets = torch.tensor([0, words - 1, words // 2, -1, words - 300], device=gpu)
    x = (torch.randn(5, width, generator=g, device=gpu) +
         3.0 * table[targets.clamp(min=0)].float()).bfloat16()
    xd, td = x.requires_grad_(), table.requires_grad_()
    dloss = torch.rand(5, generator=g, device=gpu)
    loss = nacho_amd.gpu_linear_cross_entropy(xd, td, targets, reduction="none")
    dx, dtable = torch.autograd.grad(loss, (xd, td), dloss)
    z = x.detach().double() @ table.detach().double().T
    lse = torch.logsumexp(z, 1)
    held = targets >= 0
    at = targets.clamp(min=0)[:, None]
    # logits of about 1 with products of 8192: their sums' error, in float32, is far below 1e-4
    each = torch.where(held, lse - z.gather(1, at)[:, 0], 0.0)
    assert float((loss.double() - each).abs().max()) < 1e-4
    dz = torch.exp(z - lse[:, None]).scatter_add_(1, at, torch.full_like(at, -1).double())
    dz *= torch.where(held, dloss, 0.0).double()[:, None]
    # bfloat16: dz is rounded, and the result
    u = 2.0 ** -8
    right = dz.T @ x.detach().double()
    off = (2 * u + 1e-4) * (dz.abs().T @ x.detach().double().abs())
    assert ((dtable.double() - right).abs() <= off + 1e-30).all()
    del right, off, dtable
    w = table.detach().double()
    off = (2 * u + 1e-4) * (dz.abs() @ w.abs())
    assert ((dx.double() - dz @ w).abs() <= off + 1e-30).all()


def test_loss_of_more_tokens_than_a_launch_has_workgroups(gpu):
    tokens, some, words, width = (1 << 26) + 8, 300, 5, 8  # four wavefronts of a workgroup have one each
    g = torch.Generator(device=gpu).manual_seed(3)
    few = torch.randn(some, width, generator=g, device=gpu).bfloat16()
    table = torch.randn(words, width, generator=g, device=gpu).bfloat16()
    few_targets = torch.randint(-1, words, (some,), generator=g, device=gpu)
    # (copies: torch's index of so many rows has the same fault that is looked for here)
    x = few.repeat(tokens // some + 1, 1)[:tokens]
    targets = few_targets.repeat(tokens // some + 1)[:tokens]
    assert torch.equal(x[-1], few[(tokens - 1) % some])
    want = Loss(few, table, few_targets, reduction="none", dloss=torch.ones(some, device=gpu))
    loss, stats = nacho_amd.gpu_linear_cross_entropy(x, table, targets, reduction="none",
                                                     return_stats=True)

    def repeated(got, right, off):
        """Rows that come again and again, in parts of which each is the same."""
        whole = tokens // some * some
        got = got.reshape(tokens, -1)
        first = got[:some]
        near(first, right.reshape(some, -1), off.reshape(some, -1))
        assert torch.equal(got[:whole].view(-1, some, got.shape[1]),
                           first.expand(tokens // some, -1, -1))
        assert torch.equal(got[whole:], first[:tokens - whole])

    repeated(loss, want.each, want.each_off)
    dloss = torch.ones(tokens, device=gpu)
    dx, dtable = nacho_amd.gpu_linear_cross_entropy_backward(dloss, x, table, targets, stats,
                                                             reduction="none")
    # (dz of many tokens is rounded; this many are not in two parts)
    u = 2.0 ** -8
    held = (few_targets >= 0)[:, None]
    z = few.double() @ table.double().T
    dz = torch.softmax(z, -1).scatter_add_(1, few_targets.clamp(min=0)[:, None],
                                           torch.full((some, 1), -1.0, device=gpu).double())
    dz = torch.where(held, dz, 0.0)
    repeated(dx, want.dx, want.dx_off + u * (dz.abs() @ table.double().abs()).view_as(want.dx))
    # Tokens are summed in at most 64 splits of 2^20 and a few, the splits' sums one by one: no more
    # than 2^20 + 1000 roundings; and dz's and the result's.
    times = (tokens // some + (torch.arange(some, device=gpu) < tokens % some)).double()[:, None]
    right = (dz * times).T @ few.double()
    size = (dz.abs() * times).T @ few.double().abs()
    off = ((1 << 20) + 1000) * 2.0 ** -24 * size + u * size + u * right.abs()
    assert ((dtable.double() - right).abs() <= off).all()


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16), ids=str)
def test_sums_over_many_tokens_are_summed_in_parts(gpu, dtype):
    """dtable's sums over 1,000,003 tokens are 64 sums of at most 15,680 products, which are added: no more
    than 15,680 + 64 roundings of their terms' magnitudes, 9.4e-4, where one sum has a million."""
    tokens, words, width = 1_000_003, 40, 16
    g = torch.Generator(device=gpu).manual_seed(4)
    x = (1.0 + torch.rand(tokens, width, generator=g, device=gpu)).to(dtype)
    table = (0.1 * torch.randn(words, width, generator=g, device=gpu)).to(dtype)
    targets = torch.randint(-1, words, (tokens,), generator=g, device=gpu)
    stats = nacho_amd.gpu_linear_cross_entropy(x, table, targets, reduction="sum",
                                               return_stats=True)[1]
    dloss = torch.tensor(1e-3, device=gpu)
    got = nacho_amd.gpu_linear_cross_entropy_backward(dloss, x, table, targets, stats,
                                                      reduction="sum")[1]
    want = Loss(x, table, targets, reduction="sum", dloss=dloss)
    held = (targets >= 0)[:, None]
    dz = torch.softmax(x.double() @ table.double().T, -1)
    dz.scatter_add_(1, targets.clamp(min=0)[:, None], torch.full((tokens, 1), -1.0, device=gpu).double())
    size = (torch.where(held, dz, 0.0).abs() * float(dloss)).T @ x.double()
    one_sum = (2 * int(held.sum()) + 4) * 2.0 ** -24
    parts = (15_680 + 64 + 4) * 2.0 ** -24
    near(got, want.dtable, want.dtable_off + (parts - one_sum) * size, "dtable")
