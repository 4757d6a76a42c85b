"""A training step's ends together, as a model uses them: words to rows and, through a layer, to a loss
against a table that is also the embedding's, the gradients clipped into float32 copies."""

import pytest
import torch

import nacho_amd
from tests.loss_reference import Loss, near

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


def _step(ids, targets, table, layer, scale):
    """Loss, gradients, their norm and the clipped float32 copies."""
    rows = nacho_amd.gpu_embedding(ids, table, scale=scale)
    hidden = rows * layer
    loss = nacho_amd.gpu_linear_cross_entropy(hidden, table, targets, scale=1.0 / scale)
    grads = torch.autograd.grad(loss, (table, layer))
    masters = [torch.empty(g.shape, device=g.device) for g in grads]
    norm = nacho_amd.gpu_clip_grad_norm(grads, 0.01, out=masters)
    return loss.detach(), grads, norm, masters


@pytest.mark.parametrize("sizes", ((1, 5, 8), (40, 300, 64), (300, 1000, 104)), ids=str)
def test_step(gpu, sizes):
    """In float32, against autograd in float64.  The table's two gradients meet in one."""
    tokens, words, width = sizes
    g = torch.Generator(device=gpu).manual_seed(1)
    normal = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
    ids = torch.randint(0, words, (tokens,), generator=g, device=gpu)
    targets = torch.randint(-1, words, (tokens,), generator=g, device=gpu)
    targets[0] = 0
    table = (normal(words, width) * width ** -0.5).requires_grad_()
    layer = normal(width).requires_grad_()
    scale = width ** 0.5
    loss, grads, norm, masters = _step(ids, targets, table, layer, scale)

    t64, l64 = (x.detach().double().requires_grad_() for x in (table, layer))
    hidden = t64[ids] * scale * l64
    z = hidden @ t64.T / scale
    want = torch.nn.functional.cross_entropy(z, torch.where(targets < 0, -100, targets))
    exact = torch.autograd.grad(want, (t64, l64))
    # Sums of at most `words` and `tokens` products, an exponent's error among them: in proportion
    # to the largest entry of each gradient, a few hundred roundings.
    size = 4 * (tokens + words + width + 64) * E
    assert abs(float(loss) - float(want)) <= size * (1 + abs(float(want)))
    for got, right in zip(grads, exact):
        assert float((got.double() - right).abs().max()) <= size * float(right.abs().max()) + 1e-12
    total = float(sum(x.double().square().sum() for x in grads)) ** 0.5
    assert abs(float(norm) - total) <= 2 * E * total
    factor = min(1.0, 0.01 / (total + 1e-6))
    for got, m in zip(grads, masters):
        assert ((m.double() - got.double() * factor).abs() <= 3 * E * m.double().abs()).all()


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16), ids=str)
def test_loss_of_looked_up_rows(gpu, dtype):
    """16-bit rows straight from the table to the loss, padding on both sides."""
    g = torch.Generator(device=gpu).manual_seed(2)
    table = (torch.randn(700, 72, generator=g, device=gpu) * 0.2).to(dtype).requires_grad_()
    ids = torch.randint(-1, 700, (6, 50), generator=g, device=gpu)
    targets = torch.randint(-1, 700, (6, 50), generator=g, device=gpu)
    rows = nacho_amd.gpu_embedding(ids, table, scale=2.0)
    loss = nacho_amd.gpu_linear_cross_entropy(rows, table, targets)
    drows, dtable = torch.autograd.grad(loss, (rows, table), retain_graph=True)
    want = Loss(rows, table, targets, dloss=torch.ones((), device=gpu))
    near(loss, want.loss, want.loss_off, "loss")
    near(drows, want.dx, want.dx_off, "drows")
    back = nacho_amd.gpu_embedding_backward(drows, ids, 700, scale=2.0)
    direct, = torch.autograd.grad(nacho_amd.gpu_embedding(ids, table, scale=2.0), table, drows)
    assert torch.equal(back, direct)
    # autograd adds the table's two gradients in its type
    alone, = torch.autograd.grad(nacho_amd.gpu_linear_cross_entropy(rows.detach(), table, targets),
                                 table)
    assert torch.equal(dtable, alone + back)


def test_graph_replays(gpu):
    """The whole step in one graph, replayed on other words between eager steps."""
    table = torch.randn(500, 64, device=gpu).bfloat16() * 0.3
    ids = torch.randint(0, 500, (400,), device=gpu)
    targets = torch.randint(-1, 500, (400,), device=gpu)
    one = torch.ones((), device=gpu)
    outs = [torch.empty(500, 64, device=gpu) for _ in range(2)]

    def step():
        rows = nacho_amd.gpu_embedding(ids, table, scale=2.0)
        loss, stats = nacho_amd.gpu_linear_cross_entropy(rows, table, targets, return_stats=True)
        drows, dhead = nacho_amd.gpu_linear_cross_entropy_backward(one, rows, table, targets, stats)
        dwords = nacho_amd.gpu_embedding_backward(drows, ids, 500, scale=2.0)
        norm = nacho_amd.gpu_clip_grad_norm([dhead, dwords], 0.1, out=outs)
        return loss, norm, outs[0], outs[1]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for _ in range(2):  # two graphs of the same step, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step())
        graphs.append(graph)
    for i in range(6):
        ids.random_(0, 500)
        targets.random_(-1, 500)
        table.normal_().mul_(0.3)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in results[i % 2]]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
