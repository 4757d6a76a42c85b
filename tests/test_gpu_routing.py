"""Tokens sorted by expert and back, with their gradients, against plain float64 loops."""

import pytest
import torch

import nacho_amd

pytestmark = pytest.mark.gpu

ROUNDOFF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E = 2.0 ** -24
TYPES = tuple(ROUNDOFF)

# tokens, per_token, experts, share of dropped choices
CHOICES = [(1, 1, 1, 0.0), (5, 2, 4, 0.0), (48, 2, 16, 0.1), (300, 3, 7, 0.5), (1000, 4, 60, 0.05),
           (1025, 4, 100, 0.0), (3001, 8, 256, 0.02), (20000, 1, 2048, 0.0), (700, 6, 1, 0.2),
           (40, 2, 3, 1.0), (16400, 4, 64, 0.0)]


def _choices(seed, tokens, per_token, experts, dropped, dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    x = (torch.rand(tokens, per_token, generator=g) ** 2 * experts).to(dtype)
    out = torch.rand(tokens, per_token, generator=g) < dropped
    bad = torch.where(torch.rand(tokens, per_token, generator=g) < 0.5, -1, experts + 3).to(dtype)
    return torch.where(out, bad, x)


def _plain(choices, experts):
    flat = choices.reshape(-1).tolist()
    there = [e for e, x in enumerate(flat) if 0 <= x < experts]
    order = sorted(there, key=lambda e: (flat[e], e))
    pos = [0]
    for x in range(experts):
        pos.append(pos[-1])
    for e in there:
        pos[flat[e] + 1] += 1
    for x in range(experts):
        pos[x + 1] += pos[x]
    slot = torch.full((len(flat),), -1, dtype=torch.int32)
    slot[torch.tensor(order, dtype=torch.long)] = torch.arange(len(order), dtype=torch.int32)
    behind = [e for e in range(len(flat)) if not 0 <= flat[e] < experts]
    return (torch.tensor(pos, dtype=torch.int32),
            torch.tensor(order + behind, dtype=torch.int32), slot.view(choices.shape))


@pytest.mark.parametrize("ids", (torch.int32, torch.int64), ids=str)
@pytest.mark.parametrize("sizes", CHOICES, ids=str)
def test_route(gpu, sizes, ids):
    choices = _choices(1, *sizes, dtype=ids)
    if ids == torch.int64:
        choices[0, 0] += 1 << 40  # dropped: what is past 32 bits counts
    got = nacho_amd.gpu_route(choices.to(gpu), sizes[2])
    for name, want in zip(("pos", "order", "slot"), _plain(choices, sizes[2])):
        assert torch.equal(getattr(got, name).cpu(), want), name


def test_route_without_tokens(gpu):
    route = nacho_amd.gpu_route(torch.zeros(0, 2, dtype=torch.int32, device=gpu), 5)
    assert not route.pos.any() and route.order.numel() == 0
    x = torch.zeros(0, 16, device=gpu, requires_grad=True)
    rows = nacho_amd.gpu_dispatch(x, route)
    out = nacho_amd.gpu_combine(rows, route, torch.zeros(0, 2, device=gpu))
    assert rows.shape == out.shape == (0, 16)
    assert torch.autograd.grad(out.sum(), x)[0].shape == (0, 16)


def _near(got, want, off, what):
    over = (got.detach().double().cpu() - want).abs() - off
    assert not torch.isnan(over).any(), what
    assert over.numel() == 0 or float(over.max()) <= 0.0, f"{what}: {float(over.max())} past"


def _check_rows(gpu, sizes, width, dtype, make=lambda x: x):
    """dispatch, combine and their gradients; `make` changes the operands' layout."""
    tokens, k, experts, _ = sizes
    choices = _choices(2, *sizes)
    pos, order, slot = _plain(choices, experts)
    held = int(pos[-1])
    g = torch.Generator().manual_seed(3)
    normal = lambda n: torch.randn(n, width, generator=g).to(dtype)  # noqa: E731
    x, y, dout, drows = normal(tokens), normal(tokens * k), normal(tokens), normal(tokens * k)
    y[held:] = float("nan")  # never read
    drows[held:] = float("nan")
    w = torch.rand(tokens, k, generator=g)
    u = ROUNDOFF[dtype]

    route = nacho_amd.gpu_route(choices.to(gpu), experts)
    xd, yd = (make(t.to(gpu)).requires_grad_() for t in (x, y))
    wd = w.to(gpu).requires_grad_()
    rows = nacho_amd.gpu_dispatch(xd, route)
    token = order[:held].long() // k
    want = torch.zeros(tokens * k, width, dtype=dtype)
    want[:held] = x[token]
    assert torch.equal(rows.cpu(), want)

    out = nacho_amd.gpu_combine(yd, route, wd)
    flat = w.double().reshape(-1)[order[:held].long()][:, None]
    terms = y[:held].double() * flat
    want = torch.zeros(tokens, width, dtype=torch.float64).index_add_(0, token, terms)
    size = torch.zeros_like(want).index_add_(0, token, terms.abs())
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
    _near(out, want, 1.01 * (u * want.abs() + (k + 1) * E * size) + tiny, "out")

    dx, = torch.autograd.grad(rows, xd, make(drows.to(gpu)))
    terms = drows[:held].double()
    want = torch.zeros(tokens, width, dtype=torch.float64).index_add_(0, token, terms)
    size = torch.zeros_like(want).index_add_(0, token, terms.abs())
    _near(dx, want, 1.01 * (u * want.abs() + k * E * size) + tiny, "dx")

    dy, dw = torch.autograd.grad(out, (yd, wd), make(dout.to(gpu)))
    want = torch.zeros(tokens * k, width, dtype=torch.float64)
    want[:held] = dout.double()[token] * flat
    _near(dy, want, 1.01 * (u + E) * want.abs() + tiny, "dy")
    both = dout.double()[token] * y[:held].double()
    want = torch.zeros(tokens * k, dtype=torch.float64)
    want[order[:held].long()] = both.sum(-1)
    size = torch.zeros(tokens * k, dtype=torch.float64)
    size[order[:held].long()] = both.abs().sum(-1)
    _near(dw, want.view(tokens, k), 1.01 * (width + 1) * E * size.view(tokens, k), "dw")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width", (1, 7, 8, 64, 200, 1000, 4096, 5001))
def test_widths(gpu, width, dtype):
    _check_rows(gpu, (53, 3, 9, 0.1), width, dtype)


@pytest.mark.parametrize("sizes", CHOICES, ids=str)
def test_sizes(gpu, sizes):
    _check_rows(gpu, sizes, 64, torch.bfloat16)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layouts(gpu, dtype):
    """Rows of wider matrices, rows that start between 16-byte pieces, and columns."""
    def sliced(by):
        def make(x):
            big = torch.full((x.shape[0] + 1, x.shape[1] + by), float("nan"), dtype=x.dtype,
                             device=x.device)
            big[1:, by // 2:by // 2 + x.shape[1]] = x
            return big[1:, by // 2:by // 2 + x.shape[1]].detach()
        return make

    for make in (sliced(16), sliced(6), lambda x: x.t().contiguous().t()):
        _check_rows(gpu, (53, 3, 9, 0.1), 64, dtype, make)


def test_broadcast_gradients(gpu):
    route = nacho_amd.gpu_route(_choices(4, 30, 2, 5, 0.0).to(gpu), 5)
    x = torch.randn(30, 24, device=gpu, requires_grad=True)
    nacho_amd.gpu_dispatch(x, route).sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2.0))
    y = torch.randn(60, 24, device=gpu, requires_grad=True)
    w = torch.ones(30, 2, device=gpu, requires_grad=True)
    nacho_amd.gpu_combine(y, route, w).sum().backward()
    assert torch.equal(y.grad, torch.ones_like(y))


def test_weights_of_another_type(gpu):
    route = nacho_amd.gpu_route(_choices(5, 30, 2, 5, 0.0).to(gpu), 5)
    y = torch.randn(60, 24, device=gpu)
    w = torch.rand(30, 2, device=gpu).bfloat16().requires_grad_()
    out = nacho_amd.gpu_combine(y, route, w)
    assert torch.equal(out, nacho_amd.gpu_combine(y, route, w.float()))
    assert torch.autograd.grad(out.sum(), w)[0].dtype == torch.bfloat16


def test_gradient_against_differences(gpu):
    """Directional slopes of the float64 definition, which is linear in rows and in weights."""
    sizes = (40, 3, 6, 0.1)
    choices = _choices(6, *sizes)
    pos, order, slot = _plain(choices, 6)
    held, token = int(pos[-1]), None
    token = order[:held].long() // 3
    g = torch.Generator().manual_seed(7)
    y, dout = torch.randn(120, 16, generator=g), torch.randn(40, 16, generator=g)
    w = torch.rand(40, 3, generator=g)

    def value(y, w):
        terms = y[:held] * w.reshape(-1)[order[:held].long()][:, None]
        out = torch.zeros(40, 16, dtype=torch.float64).index_add_(0, token, terms)
        return float((out * dout.double()).sum())

    route = nacho_amd.gpu_route(choices.to(gpu), 6)
    yd, wd = y.to(gpu).requires_grad_(), w.to(gpu).requires_grad_()
    grads = torch.autograd.grad(nacho_amd.gpu_combine(yd, route, wd), (yd, wd), dout.to(gpu))
    ops = [y.double(), w.double()]
    for i in range(2):
        step = torch.randn(ops[i].shape, generator=g, dtype=torch.float64)
        up, down = list(ops), list(ops)
        up[i], down[i] = ops[i] + step, ops[i] - step
        slope = (value(*up) - value(*down)) / 2
        got = float((grads[i].double().cpu() * step).sum())
        assert abs(got - slope) <= 20 * E * float((grads[i].double().cpu() * step).abs().sum())


def test_csr(gpu):
    """A route as an operand of the sparse entry points: experts x tokens."""
    choices = torch.tensor([[0, 2], [2, 1], [5, 0], [1, 2]], dtype=torch.int32)
    w = torch.arange(8, dtype=torch.float32).view(4, 2) + 1
    route = nacho_amd.gpu_route(choices.to(gpu), 3)
    a = route.csr(w.to(gpu))
    nacho_amd.validate_csr(a)
    dense = torch.zeros(3, 4)
    for t in range(4):
        for i in range(2):
            if choices[t, i] < 3:
                dense[choices[t, i], t] = w[t, i]
    z = nacho_amd.gpu_csr_add_f32(a, a)
    got = torch.sparse_csr_tensor(z.dim_j_offsets.long(), z.dim_j_indices.long(), z.values,
                                  (3, 4)).to_dense().cpu()
    assert torch.equal(got, 2 * dense)


def test_graph_replays(gpu):
    choices = _choices(8, 3000, 4, 40, 0.05).to(gpu)
    x, w = torch.randn(3000, 64, device=gpu), torch.rand(3000, 4, device=gpu)

    def step():
        route = nacho_amd.gpu_route(choices, 40)
        rows = nacho_amd.gpu_dispatch(x, route)
        return route.slot, rows, nacho_amd.gpu_combine(rows, route, w)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        x.normal_()
        choices.copy_(_choices(9 + i, 3000, 4, 40, 0.05))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_refusals(gpu):
    choices = _choices(1, 10, 2, 4, 0.0).to(gpu)
    route = nacho_amd.gpu_route(choices, 4)
    x, w = torch.zeros(10, 8, device=gpu), torch.zeros(10, 2, device=gpu)
    for call, error, text in [
            (lambda: nacho_amd.gpu_route(choices.cpu(), 4), ValueError, "GPU tensor"),
            (lambda: nacho_amd.gpu_route(choices.float(), 4), TypeError, "experts"),
            (lambda: nacho_amd.gpu_route(choices[0], 4), ValueError, "dimensions"),
            (lambda: nacho_amd.gpu_route(choices, 0), ValueError, "n_experts"),
            (lambda: nacho_amd.gpu_route(choices, 2049), ValueError, "n_experts"),
            (lambda: nacho_amd.gpu_route(choices[:, :0], 4), ValueError, "at least one"),
            (lambda: nacho_amd.gpu_dispatch(x, choices), TypeError, "Route"),
            (lambda: nacho_amd.gpu_dispatch(x[1:], route), ValueError, "10 rows"),
            (lambda: nacho_amd.gpu_dispatch(x.double(), route), TypeError, "x: expected"),
            (lambda: nacho_amd.gpu_dispatch(x.cpu(), route), ValueError, "GPU tensor"),
            (lambda: nacho_amd.gpu_combine(x, route, w), ValueError, "20 rows"),
            (lambda: nacho_amd.gpu_combine(x.repeat(2, 1), route, w[1:]), ValueError, "weights"),
            (lambda: nacho_amd.gpu_combine(x.repeat(2, 1), route, w.long()), TypeError,
             "weights")]:
        with pytest.raises(error, match=text):
            call()
