"""The linear cross entropy and its gradients against their formulas in float64."""

import pytest
import torch

import nacho_amd
from tests.loss_reference import Loss, near

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.float16, torch.bfloat16)
# tokens, words, width
SIZES = [(1, 1, 1), (1, 5, 8), (2, 1, 64), (3, 100, 64), (16, 257, 72), (17, 300, 40),
         (65, 513, 136), (128, 256, 64), (129, 700, 264), (300, 1000, 104), (700, 2300, 520),
         (450, 300, 776), (321, 66000, 24), (1100, 1025, 328), (260, 20, 1032), (180, 600, 192),
         (3000, 300, 72), (9000, 1000, 40), (20000, 50, 16), (600, 700, 333)]


def _operands(gpu, seed, tokens, words, width, dtype, left=0.2, ids=torch.int64, lean=4.0):
    """Rows that lean towards their targets; some targets are none, and their rows no numbers."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
    table = (normal(words, width) * width ** -0.5).to(dtype)
    targets = torch.randint(0, words, (tokens,), generator=g, device=gpu).to(ids)
    x = normal(tokens, width) + lean * torch.rand(tokens, 1, generator=g, device=gpu) * \
        table[targets.long()].float()
    x = x.to(dtype)
    none = torch.rand(tokens, generator=g, device=gpu) < left
    bad = torch.where(torch.rand(tokens, generator=g, device=gpu) < 0.5, -100, words)
    targets = torch.where(none, bad.to(ids), targets)
    x[none] = float("nan")
    return x, table, targets


def _dloss(gpu, reduction, shape):
    if reduction != "none":
        return torch.tensor(0.7, device=gpu)
    return torch.linspace(-1.0, 2.0, max(1, shape.numel()), device=gpu)[:shape.numel()].view(shape)


def _check(gpu, x, table, targets, scale=1.0, reduction="mean", dloss=None):
    xd, td = x.detach().requires_grad_(), table.detach().requires_grad_()
    loss, stats = nacho_amd.gpu_linear_cross_entropy(xd, td, targets, scale=scale,
                                                     reduction=reduction, return_stats=True)
    dloss = _dloss(gpu, reduction, targets.shape) if dloss is None else dloss
    want = Loss(x, table, targets, scale, reduction, dloss)
    near(loss, want.loss, want.loss_off, "loss")
    held = (targets.reshape(-1) >= 0) & (targets.reshape(-1) < table.shape[0])
    lse = stats[0].double() + torch.log(stats[1].double())
    near(lse[held], want.lse[held], want.lse_off[held], "lse")
    assert not lse[~held].any()
    dx, dtable = torch.autograd.grad(loss, (xd, td), dloss)
    near(dx, want.dx, want.dx_off, "dx")
    near(dtable, want.dtable, want.dtable_off, "dtable")
    assert not dx.reshape(-1, x.shape[-1])[~held].any()
    plain = nacho_amd.gpu_linear_cross_entropy(x, table, targets, scale=scale, reduction=reduction)
    assert torch.equal(plain, loss.detach())
    again = nacho_amd.gpu_linear_cross_entropy_backward(dloss, x, table, targets, stats,
                                                        scale=scale, reduction=reduction)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dtable)
    return want


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_sizes(gpu, sizes, dtype):
    _check(gpu, *_operands(gpu, 1, *sizes, dtype))


@pytest.mark.parametrize("reduction", ("none", "mean", "sum"))
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_reductions(gpu, dtype, reduction):
    _check(gpu, *_operands(gpu, 2, 90, 400, 96, dtype, ids=torch.int32), scale=0.5,
           reduction=reduction)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width", (1, 3, 7, 33, 100, 130, 257))
def test_odd_widths(gpu, width, dtype):
    _check(gpu, *_operands(gpu, 3, 37, 300, width, dtype))


@pytest.mark.parametrize("scale", (0.0, -1.5, 30.0))
def test_scales(gpu, scale):
    _check(gpu, *_operands(gpu, 4, 50, 300, 64, torch.float32), scale=scale)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_certain_tokens(gpu, dtype):
    """Probabilities next to 1 and next to 0, and logits of thousands."""
    _check(gpu, *_operands(gpu, 5, 60, 500, 64, dtype, lean=60.0))
    _check(gpu, *_operands(gpu, 6, 60, 500, 64, dtype, lean=10.0), scale=100.0)


@pytest.mark.parametrize("tokens", (1, 20, 200))
def test_no_targets(gpu, tokens):
    x, table, targets = _operands(gpu, 7, tokens, 300, 64, torch.bfloat16, left=1.1)
    for reduction in ("none", "mean", "sum"):
        _check(gpu, x, table, targets, reduction=reduction)


def test_wide_ids(gpu):
    x, table, targets = _operands(gpu, 8, 30, 300, 64, torch.bfloat16, left=0.0)
    targets[3] += 1 << 40  # what is past 32 bits counts
    targets[4] -= 1 << 32
    _check(gpu, x, table, targets)


def test_no_tokens(gpu):
    table = torch.randn(50, 16, device=gpu, requires_grad=True)
    for shape in ((0,), (3, 0)):
        x = torch.zeros(*shape, 16, device=gpu, requires_grad=True)
        targets = torch.zeros(*shape, dtype=torch.long, device=gpu)
        each = nacho_amd.gpu_linear_cross_entropy(x, table, targets, reduction="none")
        assert each.shape == targets.shape
        loss = nacho_amd.gpu_linear_cross_entropy(x, table, targets)
        assert loss.shape == () and float(loss) == 0.0
        dx, dtable = torch.autograd.grad(loss, (x, table))
        assert dx.shape == x.shape and not dtable.any()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layouts(gpu, dtype):
    """More dimensions, rows of wider matrices, rows between 16-byte pieces, columns, one row for
    all tokens."""
    x, table, targets = _operands(gpu, 9, 48, 300, 64, dtype)
    _check(gpu, x.view(4, 12, 64), table, targets.view(4, 12), reduction="none")

    def sliced(t, by):
        big = torch.full((t.shape[0] + 1, t.shape[1] + by), float("nan"), dtype=t.dtype, device=gpu)
        big[1:, by // 2:by // 2 + t.shape[1]] = t
        return big[1:, by // 2:by // 2 + t.shape[1]].detach()

    for by in (16, 6):
        _check(gpu, sliced(x, by), sliced(table, by), targets)
    _check(gpu, x.t().contiguous().t(), table.t().contiguous().t(), targets)
    _check(gpu, x.view(4, 12, 64).transpose(0, 1), table, targets.view(4, 12).t())
    row = torch.randn(1, 64, device=gpu).to(dtype)
    _check(gpu, row.expand(48, 64), table, targets)
    _check(gpu, x, table[:1].expand(5, 64), targets.clamp(max=5))


def test_one_gradient_at_a_time(gpu):
    x, table, targets = _operands(gpu, 10, 90, 400, 96, torch.bfloat16)
    both = nacho_amd.gpu_linear_cross_entropy_backward(
        torch.ones((), device=gpu), x, table, targets,
        nacho_amd.gpu_linear_cross_entropy(x, table, targets, return_stats=True)[1])
    for i in range(2):
        ops = [x.detach(), table.detach()]
        ops[i].requires_grad_()
        loss = nacho_amd.gpu_linear_cross_entropy(*ops, targets)
        assert torch.equal(torch.autograd.grad(loss, ops[i])[0], both[i])


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32), ids=str)
def test_pieces_of_the_vocabulary(gpu, dtype):
    """More words than a piece has, and a last piece of few."""
    tokens = 4500 if dtype == torch.bfloat16 else 3000
    _check(gpu, *_operands(gpu, 11, tokens, 30100 if dtype == torch.bfloat16 else 22600, 72, dtype,
                           left=0.1))


@pytest.mark.parametrize("tokens", (1, 3, 16, 40))
def test_few_tokens_of_many_words(gpu, tokens):
    """Sums over the words that are split between workgroups."""
    _check(gpu, *_operands(gpu, 12, tokens, 70001, 200, torch.bfloat16, left=0.0))


def test_small_losses_of_float16(gpu):
    """Scaled losses, and gradients of a token's loss that float16 does not hold."""
    x, table, targets = _operands(gpu, 13, 80, 900, 64, torch.float16)
    for size in (1e-6, 3e4):
        _check(gpu, x, table, targets, reduction="sum", dloss=torch.tensor(size, device=gpu))
        each = size * torch.rand(80, device=gpu)
        each[7] = 0.0
        _check(gpu, x, table, targets, reduction="none", dloss=each)
    _check(gpu, x, table, targets, reduction="none", dloss=torch.zeros(80, device=gpu))


def test_values_that_are_not_finite(gpu):
    """A token's own values reach its loss and gradient, and the table's, and no other token's."""
    x, table, targets = _operands(gpu, 14, 40, 300, 64, torch.bfloat16, left=0.0)
    want = nacho_amd.gpu_linear_cross_entropy(x, table, targets, reduction="none")
    stats = nacho_amd.gpu_linear_cross_entropy(x, table, targets, reduction="none",
                                               return_stats=True)[1]
    ones = torch.ones(40, device=gpu)
    dx = nacho_amd.gpu_linear_cross_entropy_backward(ones, x, table, targets, stats,
                                                     reduction="none")[0]
    x[5, 3] = float("nan")
    xd = x.requires_grad_()
    td = table.requires_grad_()
    loss = nacho_amd.gpu_linear_cross_entropy(xd, td, targets, reduction="none")
    got = torch.autograd.grad(loss, (xd, td), ones)
    assert torch.isnan(loss[5]) and torch.isnan(got[0][5]).all() and torch.isnan(got[1]).all()
    keep = torch.arange(40, device=gpu) != 5
    assert torch.equal(loss[keep], want[keep]) and torch.equal(got[0][keep], dx[keep])


@pytest.mark.parametrize("value", (float("nan"), float("inf"), 3.4e38))
@pytest.mark.parametrize("tokens", (20, 300))
def test_float32_next_to_values_that_are_not_finite(gpu, tokens, value):
    """Products in parts are none where an operand is not finite: those of the others stay right."""
    x, table, targets = _operands(gpu, 27, tokens, 600, 72, torch.float32, left=0.0)
    want = Loss(x, table, targets, reduction="none", dloss=torch.ones(tokens, device=gpu))
    x[7, 5] = value
    xd = x.requires_grad_()
    loss = nacho_amd.gpu_linear_cross_entropy(xd, table, targets, reduction="none")
    dx, = torch.autograd.grad(loss, xd, torch.ones(tokens, device=gpu))
    keep = torch.arange(tokens, device=gpu) != 7
    near(loss[keep], want.loss[keep], want.loss_off[keep], "loss")
    near(dx[keep], want.dx[keep], want.dx_off[keep], "dx")
    assert not torch.isfinite(loss[7]) or abs(value) < float("inf")


@pytest.mark.parametrize("size", (2.0 ** -60, 2.0 ** 60, 2.0 ** 100))
def test_float32_of_all_sizes(gpu, size):
    x, table, targets = _operands(gpu, 28, 40, 300, 64, torch.float32, left=0.0)
    dloss = _dloss(gpu, "mean", targets.shape)
    want = Loss(x, table, targets, dloss=dloss)
    xd, td = (x * size).requires_grad_(), (table / size).requires_grad_()
    loss = nacho_amd.gpu_linear_cross_entropy(xd, td, targets)
    dx, dtable = torch.autograd.grad(loss, (xd, td), dloss)
    near(loss, want.loss, want.loss_off, "loss")
    near(dx * size, want.dx, want.dx_off, "dx")
    near(dtable / size, want.dtable, want.dtable_off, "dtable")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gradients_of_losses_that_are_not_finite(gpu, dtype):
    """They reach their own token's dx and the whole dtable, and no other token's dx."""
    x, table, targets = _operands(gpu, 29, 50, 300, 64, dtype, left=0.0)
    stats = nacho_amd.gpu_linear_cross_entropy(x, table, targets, reduction="none",
                                               return_stats=True)[1]
    dloss = 1000.0 * torch.rand(50, device=gpu) + 1.0
    want = Loss(x, table, targets, reduction="none", dloss=dloss)
    for value in (float("inf"), float("nan")):
        c = dloss.clone()
        c[9] = value
        dx, dtable = nacho_amd.gpu_linear_cross_entropy_backward(c, x, table, targets, stats,
                                                                 reduction="none")
        keep = torch.arange(50, device=gpu) != 9
        near(dx[keep], want.dx[keep], want.dx_off[keep], "dx")
        assert not torch.isfinite(dx[9]).any() and not torch.isfinite(dtable[targets[9]]).any()


def test_words_of_minus_infinity(gpu):
    """A word whose logits are all minus infinity has probability 0."""
    x = torch.ones(20, 32, device=gpu)
    table = torch.randn(300, 32, device=gpu)
    targets = torch.arange(20, device=gpu)
    want = nacho_amd.gpu_linear_cross_entropy(x, table, targets, reduction="none")
    more = torch.cat((table, torch.full((300, 32), -float("inf"), device=gpu)))
    got = nacho_amd.gpu_linear_cross_entropy(x, more, targets, reduction="none")
    assert torch.allclose(got, want, rtol=0, atol=1e-5)


def test_gradient_against_differences(gpu):
    x, table, targets = _operands(gpu, 15, 30, 200, 48, torch.float32, left=0.1)
    x = torch.where(torch.isnan(x), 0.0, x)
    g = torch.Generator(device=gpu).manual_seed(16)
    xd, td = x.requires_grad_(), table.requires_grad_()
    loss = nacho_amd.gpu_linear_cross_entropy(xd, td, targets, scale=0.7)
    grads = torch.autograd.grad(loss, (xd, td))
    ops = [x.detach().double(), table.detach().double()]
    held = targets.ge(0) & targets.lt(200)

    def value(x, table):
        z = (x @ table.T * float(torch.tensor(0.7)))[held]
        return float((torch.logsumexp(z, -1) - z.gather(1, targets[held][:, None])[:, 0]).mean())

    for i in range(2):
        step = torch.randn(ops[i].shape, generator=g, device=gpu, dtype=torch.float64)
        h = 1e-4
        up, down = list(ops), list(ops)
        up[i], down[i] = ops[i] + h * step, ops[i] - h * step
        slope = (value(*up) - value(*down)) / (2 * h)
        got = float((grads[i].double() * step).sum())
        size = float((grads[i].double() * step).abs().sum())
        # h^2 of the third derivative, at most the cube of a logit's change
        assert abs(got - slope) <= 1e-5 * size + 1e-6


def test_other_streams(gpu):
    x, table, targets = _operands(gpu, 17, 300, 3000, 128, torch.bfloat16)
    x, table = torch.where(torch.isnan(x), 0.0, x).requires_grad_(), table.requires_grad_()

    def step():
        loss = nacho_amd.gpu_linear_cross_entropy(x, table, targets)
        return loss.detach(), *torch.autograd.grad(loss, (x, table))

    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:  # two calls at once
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, want))


def test_graph_replays(gpu):
    x, table, targets = _operands(gpu, 18, 500, 2000, 96, torch.bfloat16)
    one = torch.ones((), device=gpu)

    def step():
        loss, stats = nacho_amd.gpu_linear_cross_entropy(x, table, targets, return_stats=True)
        return loss, *nacho_amd.gpu_linear_cross_entropy_backward(one, x, table, targets, stats)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        for t, new in zip((x, table, targets), _operands(gpu, 19 + i, 500, 2000, 96,
                                                         torch.bfloat16, left=0.3 * i)):
            t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_written_operands_are_noticed(gpu):
    x, table, targets = _operands(gpu, 23, 20, 50, 16, torch.float32, left=0.0)
    x.requires_grad_()
    loss = nacho_amd.gpu_linear_cross_entropy(x, table, targets)
    targets.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_refuses_tangents(gpu):
    from torch.autograd import forward_ad

    x, table, targets = _operands(gpu, 24, 5, 50, 16, torch.float32, left=0.0)
    with forward_ad.dual_level():
        for i in range(2):
            ops = [x, table]
            ops[i] = forward_ad.make_dual(ops[i], torch.ones_like(ops[i]))
            with pytest.raises(NotImplementedError, match="jvp"):
                nacho_amd.gpu_linear_cross_entropy(*ops, targets)


def test_inference_mode(gpu):
    x, table, targets = _operands(gpu, 25, 20, 50, 16, torch.float32)
    want = nacho_amd.gpu_linear_cross_entropy(x, table, targets)
    with torch.inference_mode():
        inside = targets.clone()
        assert torch.equal(nacho_amd.gpu_linear_cross_entropy(x, table, inside), want)
    x = x.requires_grad_()
    loss = nacho_amd.gpu_linear_cross_entropy(x, table, inside)
    assert torch.equal(loss.detach(), want)
    loss.backward()


def test_refusals(gpu):
    x, table, targets = _operands(gpu, 26, 10, 30, 16, torch.float32)
    f = nacho_amd.gpu_linear_cross_entropy
    b = nacho_amd.gpu_linear_cross_entropy_backward
    stats = f(x, table, targets, return_stats=True)[1]
    one = torch.ones((), device=gpu)
    for call, error, text in [
            (lambda: f(x.cpu(), table, targets), ValueError, "x: expected a GPU tensor"),
            (lambda: f(x, table.cpu(), targets), ValueError, "table: expected a GPU tensor"),
            (lambda: f(x, table, targets.cpu()), ValueError, "targets: expected a GPU tensor"),
            (lambda: f(x.double(), table, targets), TypeError, "x: expected dtype"),
            (lambda: f(x.half(), table, targets), TypeError, "table: expected dtype"),
            (lambda: f(x, table, targets.float()), TypeError, "targets: expected dtype"),
            (lambda: f(x, table[:, :8], targets), ValueError, "rows of 8"),
            (lambda: f(x, table[0], targets), ValueError, "table: expected 2 dimensions"),
            (lambda: f(x, table[:0], targets), ValueError, "table: expected words"),
            (lambda: f(x, table, targets[1:]), ValueError, "targets: expected shape"),
            (lambda: f(x[0], table, targets), ValueError, "targets: expected shape"),
            (lambda: f(x, table, targets, scale=float("nan")), ValueError, "scale"),
            (lambda: f(x, table, targets, scale=1e39), ValueError, "scale"),
            (lambda: f(x, table, targets, reduction="max"), ValueError, "reduction"),
            (lambda: b(one.double(), x, table, targets, stats), TypeError, "dloss"),
            (lambda: b(one[None], x, table, targets, stats), ValueError, "dloss: expected shape"),
            (lambda: b(one, x, table, targets, stats[:1]), ValueError, "stats: expected shape"),
            (lambda: b(one, x, table, targets, stats, reduction="none"), ValueError, "dloss")]:
        with pytest.raises(error, match=text):
            call()


@pytest.mark.parametrize("tokens", [1, 9, 16])
def test_few_float32_tokens_sum_wide_rows_in_steps(gpu, tokens):
    """Logits of few float32 tokens are summed over 32 columns at a time, and these sums added: for
    D columns 32 + D / 32 roundings, each at most 2^-24 of a sum of terms of one sign.

    All terms are c = 1 + 0.9 2^-13.  In one sum of all the last 8192 terms each lose 0.9 2^-13, one
    by one or four together (sums from 2^13 on are multiples of 2^-10): 0.9 of 16386, 5.5e-5, where
    32 + 512 roundings are at most 3.3e-5."""
    width, scale = 16384, 2.0 ** -14
    x = torch.ones(tokens, width, device=gpu)
    table = torch.zeros(3, width, device=gpu)
    table[1] = 1 + 0.9 * 2.0 ** -13
    targets = torch.ones(tokens, dtype=torch.int64, device=gpu)
    _, stats = nacho_amd.gpu_linear_cross_entropy(x, table, targets, scale=scale,
                                                  return_stats=True)
    exact = table[1].double().sum().item() * scale
    # (the multiplication by the scale is exact)
    assert (stats[0].double() - exact).abs().max().item() <= (32 + width // 32) * 2.0 ** -24 * exact
