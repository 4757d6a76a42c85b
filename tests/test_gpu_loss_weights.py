"""Gradients of the linear cross entropy where tokens count differently: weights of
every size, few targets among many tokens, no target at all; and that nothing in them comes from
scratch memory."""

import pytest
import torch

import nacho_amd
from tests.loss_reference import TINY, Loss, near

pytestmark = pytest.mark.gpu

HALVES = (torch.float16, torch.bfloat16)


def _operands(gpu, seed, tokens, words, width, dtype, lean=4.0):
    """Rows that lean towards their targets."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
    table = (normal(words, width) * width ** -0.5).to(dtype)
    targets = torch.randint(0, words, (tokens,), generator=g, device=gpu)
    x = normal(tokens, width) + lean * torch.rand(tokens, 1, generator=g, device=gpu) * \
        table[targets].float()
    return x.to(dtype), table, targets


def _gradients(x, table, targets, dloss, reduction="none", scale=1.0):
    stats = nacho_amd.gpu_linear_cross_entropy(x, table, targets, scale=scale, reduction=reduction,
                                               return_stats=True)[1]
    return nacho_amd.gpu_linear_cross_entropy_backward(dloss, x, table, targets, stats,
                                                       scale=scale, reduction=reduction)


def _after(value, gpu, call):
    """A call whose memory held bytes of `value` before."""
    pool = torch.cuda.MemPool()
    with torch.cuda.use_mem_pool(pool):
        block = torch.full((1 << 28,), value, dtype=torch.uint8, device=gpu)
        del block
        got = [t.cpu() for t in call()]
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("dtype", (torch.float32, *HALVES), ids=str)
@pytest.mark.parametrize("sizes", ((300, 1100, 64), (300, 600, 72), (200, 1100, 136), (30, 70, 64),
                                   (9, 300, 40), (2100, 1100, 333), (3000, 22600, 72)), ids=str)
def test_nothing_comes_from_scratch(gpu, sizes, dtype):
    """The same bits whatever the call's memory held: zeros, or bytes that are no numbers."""
    x, table, targets = _operands(gpu, 2, *sizes, dtype)
    targets[::5] = -1
    dloss = torch.rand(targets.shape, device=gpu)
    call = lambda: _gradients(x, table, targets, dloss)  # noqa: E731
    for a, b in zip(_after(0, gpu, call), _after(0xff, gpu, call)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("tokens", (40, 140, 2100))
@pytest.mark.parametrize("dtype", (torch.float32, *HALVES), ids=str)
def test_a_tokens_dx_is_as_exact_as_its_own_weight_allows(gpu, dtype, tokens):
    """Weights from 2^16 down to 2^-4 in one call, and nearly even probabilities of 2^-15: what
    another token weighs is nothing to a token's own gradient.

    A token's dx and how far it may be off are those of a weight of 1, times its own, whose product
    is rounded to the result's type."""
    words, width = 33000, 64
    g = torch.Generator(device=gpu).manual_seed(3)
    table = (0.5 + 0.1 * torch.randn(words, width, generator=g, device=gpu)).to(dtype)
    x = (0.02 * torch.randn(tokens, width, generator=g, device=gpu)).to(dtype)
    targets = torch.randint(0, words, (tokens,), generator=g, device=gpu)
    c = 2.0 ** torch.linspace(16, -4, tokens, device=gpu)
    dx, _ = _gradients(x, table, targets, c)
    one = Loss(x, table, targets, reduction="none", dloss=torch.ones(tokens, device=gpu))
    c = c.double()[:, None]
    near(dx, one.dx * c, one.dx_off * c + TINY[dtype], "dx")


@pytest.mark.parametrize("reduction", ("mean", "none"))
@pytest.mark.parametrize("held", (1, 3, 128))
@pytest.mark.parametrize("tokens", (129, 1000, 3000))
@pytest.mark.parametrize("dtype", HALVES, ids=str)
def test_few_targets_among_many_tokens(gpu, dtype, tokens, held, reduction):
    """The gradients of up to 128 tokens that have a target are as exact as those of a call that has
    these tokens alone: rounded once, for the result."""
    x, table, targets = _operands(gpu, 4, tokens, 900, 72, dtype)
    some = torch.randperm(tokens, generator=torch.Generator().manual_seed(5))[:held].sort()[0]
    some = some.to(gpu)
    left = torch.full_like(targets, -1)
    left[some] = targets[some]
    dloss = torch.rand(tokens, device=gpu) if reduction == "none" else torch.tensor(0.7, device=gpu)
    own = dloss[some] if reduction == "none" else dloss
    dx, dtable = _gradients(x, table, left, dloss, reduction)
    want = Loss(x[some], table, targets[some], 1.0, reduction, own)
    near(dx[some], want.dx, want.dx_off, "dx")
    near(dtable, want.dtable, want.dtable_off, "dtable")
    none = torch.ones(tokens, dtype=torch.bool, device=gpu)
    none[some] = False
    assert not dx[none].any()


@pytest.mark.parametrize("value", (float("inf"), float("-inf"), float("nan"), 3e38))
@pytest.mark.parametrize("dtype", (torch.float32, *HALVES), ids=str)
def test_no_target_has_no_gradient(gpu, dtype, value):
    """A sum over no tokens is 0, whatever the gradient of its result."""
    for tokens in (1, 40, 200, 3000):
        x, table, targets = _operands(gpu, 1, tokens, 300, 64, dtype)
        for reduction in ("mean", "sum", "none"):
            shape = targets.shape if reduction == "none" else ()
            dx, dtable = _gradients(x, table, torch.full_like(targets, -1),
                                    torch.full(shape, value, device=gpu), reduction)
            assert not dx.any() and not dtable.any(), (tokens, reduction)


@pytest.mark.parametrize("tokens", (50, 300))
def test_one_gradient_at_a_time(gpu, tokens):
    """float16 tokens with weights: each gradient by itself, of two dz's for both."""
    x, table, targets = _operands(gpu, 6, tokens, 700, 72, torch.float16)
    targets[::7] = -1
    c = 2.0 ** torch.linspace(-6, 6, tokens, device=gpu)
    want = Loss(x, table, targets, reduction="none", dloss=c)
    for wanted in ((True, False), (False, True), (True, True)):
        ops = [t.detach().requires_grad_(w) for t, w in zip((x, table), wanted)]
        loss = nacho_amd.gpu_linear_cross_entropy(*ops, targets, reduction="none")
        loss.backward(c)
        if wanted[0]:
            near(ops[0].grad, want.dx, want.dx_off, "dx")
        if wanted[1]:
            near(ops[1].grad, want.dtable, want.dtable_off, "dtable")


@pytest.mark.parametrize("tokens", (300, 2500))
@pytest.mark.parametrize("dtype", HALVES, ids=str)
def test_graph_replays(gpu, dtype, tokens):
    """One graph of a step whose replays have no target, few, and many: dz in two parts and in one."""
    x, table, targets = _operands(gpu, 7, tokens, 900, 72, dtype)
    c = torch.rand(tokens, device=gpu)

    def step():
        loss, stats = nacho_amd.gpu_linear_cross_entropy(x, table, targets, reduction="none",
                                                         return_stats=True)
        return loss, *nacho_amd.gpu_linear_cross_entropy_backward(c, x, table, targets, stats,
                                                                  reduction="none")

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i, held in enumerate((3, tokens, 0, 128, 129)):
        new_x, new_table, new_targets = _operands(gpu, 8 + i, tokens, 900, 72, dtype)
        new_targets[held:] = -1
        c.uniform_(0.1, 1000.0)
        for t, new in zip((x, table, targets), (new_x, new_table, new_targets)):
            t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b), held
