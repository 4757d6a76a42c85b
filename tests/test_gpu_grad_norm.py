"""The common norm of many tensors, and clipping, against plain float64 sums."""

import math

import pytest
import torch

import nacho_amd

pytestmark = pytest.mark.gpu

ROUNDOFF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E = 2.0 ** -24
TYPES = tuple(ROUNDOFF)
SIZES = [(1,), (5,), (0,), (1000,), (33, 7), (32768,), (32769,), (3, 0, 2), (300, 401), (2, 3, 5, 7)]


def _tensors(gpu, sizes, dtypes=TYPES, seed=0, size=1.0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return [(size * torch.randn(s, generator=g, device=gpu)).to(dtypes[i % len(dtypes)])
            for i, s in enumerate(sizes)]


def _norm(tensors):
    return math.sqrt(sum(float(t.double().square().sum()) for t in tensors if t is not None))


def _check(tensors, max_norm, out=None):
    """A call in place, or into `out`; tensors are as the call leaves them."""
    before = [None if t is None else t.clone() for t in tensors]
    want = _norm(tensors)
    got = nacho_amd.gpu_clip_grad_norm(tensors, max_norm, out=out)
    assert got.dtype == torch.float32 and got.shape == ()
    # (a sum's order in float64 is nothing to float32's rounding)
    assert abs(float(got) - want) <= 1.001 * E * want
    factor = 1.0 if max_norm == math.inf else min(1.0, max_norm / (want + 1e-6))
    for old, t, o in zip(before, tensors, tensors if out is None else out):
        if old is None:
            continue
        u = ROUNDOFF[o.dtype]
        exact = old.double() * factor
        tiny = 2.0 ** -25 if o.dtype == torch.float16 else 2.0 ** -126
        # the factor's rounding, the product's in float32, and the result's
        off = (u + 2.01 * E) * exact.abs() + tiny
        assert ((o.double() - exact).abs() <= 1.01 * off).all()
        if out is not None:
            assert torch.equal(t, old)
    return got


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("max_norm", (0.0, 1.0, 1e9, math.inf))
def test_in_place(gpu, dtype, max_norm):
    tensors = _tensors(gpu, SIZES, (dtype,))
    before = [t.clone() for t in tensors]
    norm = nacho_amd.gpu_grad_norm(tensors)
    assert torch.equal(_check(tensors, max_norm), norm)
    if max_norm >= 1e9:
        assert all(torch.equal(a, b) for a, b in zip(tensors, before))


@pytest.mark.parametrize("max_norm", (0.5, 1e9))
def test_into_others(gpu, max_norm):
    """Of the same types and of float32, next to each other in one buffer."""
    tensors = _tensors(gpu, SIZES)
    _check(tensors, max_norm, [torch.full_like(t, float("nan")) for t in tensors])
    for gap in (0, 1, 64):
        flat = torch.full((sum(t.numel() + gap for t in tensors),), 7.0, device=gpu)
        outs, at = [], 0
        for t in tensors:
            outs.append(flat[at:at + t.numel()].view(t.shape))
            at += t.numel() + gap
        _check(tensors, max_norm, outs)
        assert int((flat == 7.0).sum()) >= gap * len(tensors)


def test_many_tensors(gpu):
    """More than a launch's arguments hold."""
    for count in (95, 96, 97, 500):
        tensors = _tensors(gpu, [(1 + 37 * i % 1001,) for i in range(count)])
        _check(tensors, 1.0)


def test_one_tensor_and_none(gpu):
    t = torch.randn(77, device=gpu)
    want = _norm([t])
    assert abs(float(nacho_amd.gpu_grad_norm(t)) - want) <= 1.001 * E * want
    _check([None, t, None], 1.0)
    nacho_amd.gpu_clip_grad_norm(t, 0.1)
    assert abs(_norm([t]) - 0.1) < 1e-5
    empty = torch.zeros(0, device=gpu)
    assert float(nacho_amd.gpu_grad_norm([empty])) == 0.0
    assert float(nacho_amd.gpu_clip_grad_norm([empty], 1.0)) == 0.0
    assert float(nacho_amd.gpu_grad_norm(torch.zeros((), device=gpu))) == 0.0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layouts(gpu, dtype):
    """Tensors that start between 16-byte pieces, in other orders, and parts of larger ones."""
    base = torch.randn(70000, device=gpu).to(dtype)
    _check([base[1:5], base[7:9000], base[9001:60000]], 1.0)
    _check([torch.randn(40, 50, device=gpu).to(dtype).t(),
            torch.randn(4, 6, 5, device=gpu).to(dtype).permute(2, 0, 1)], 1.0)
    wide = torch.randn(40, 50, device=gpu).to(dtype)
    want = _norm([wide[:, 3:20]])
    assert abs(float(nacho_amd.gpu_grad_norm([wide[:, 3:20]])) - want) <= 1.001 * E * want
    one = torch.ones(3, 1, device=gpu).to(dtype).expand(3, 100)
    assert abs(float(nacho_amd.gpu_grad_norm(one)) - math.sqrt(300)) <= 1e-6 * 300
    for t in (wide[:, 3:20], one, wide.t()):
        _check([t], 1.0, [torch.empty(t.shape, dtype=torch.float32, device=gpu)])
    _check([wide], 1.0, [torch.empty(50, 40, dtype=dtype, device=gpu).t()])
    before = base.clone()
    _check([base[100:200]], 1.0)
    before[100:200] = base[100:200]
    assert torch.equal(base, before)


def test_sizes_of_values(gpu):
    """Squares that float32 does not hold, small tensors next to large ones, subnormal numbers."""
    for size in (1e30, 1e-30):
        _check(_tensors(gpu, [(1000,), (50,)], (torch.float32, torch.bfloat16), size=size), 1.0)
    _check([torch.full((1 << 22,), 1.0, device=gpu), torch.full((3,), 1e4, device=gpu)], 1.0)
    _check([torch.full((100,), 6e-8, device=gpu, dtype=torch.float16)], 1.0)
    _check([torch.full((100,), 6e4, device=gpu, dtype=torch.float16)], 1e9)


def test_values_that_are_not_finite(gpu):
    inf, nan = float("inf"), float("nan")
    a, b = torch.ones(100, device=gpu), torch.ones(50, device=gpu)
    a[3] = -inf
    assert float(nacho_amd.gpu_clip_grad_norm([a, b], 1.0)) == inf
    assert torch.isnan(a[3]) and not a[4:].any() and not a[:3].any() and not b.any()
    a, b = torch.ones(100, device=gpu), torch.ones(50, device=gpu)
    b[7] = nan
    assert math.isnan(float(nacho_amd.gpu_clip_grad_norm([a, b], 1.0)))
    assert torch.isnan(a).all() and torch.isnan(b).all()
    a = torch.ones(100, device=gpu)
    a[5] = inf
    assert float(nacho_amd.gpu_clip_grad_norm([a], inf)) == inf
    assert float(a[5]) == inf and float(a[6]) == 1.0


def test_a_large_tensor(gpu):
    n = (1 << 31) + 12345  # more elements than 32 bits count
    t = torch.ones(n, dtype=torch.bfloat16, device=gpu)
    assert abs(float(nacho_amd.gpu_grad_norm(t)) - math.sqrt(n)) <= E * math.sqrt(n) * 1.001
    nacho_amd.gpu_clip_grad_norm(t, 0.25 * math.sqrt(n) + 1.0)
    assert torch.equal(t[:5], t[-5:]) and abs(float(t[-1]) - 0.25) < 0.002
    assert torch.equal(t.amax(), t.amin())


def test_graph_replays(gpu):
    tensors = _tensors(gpu, [(1 + 77 * i,) for i in range(120)])
    outs = [torch.empty_like(t) for t in tensors]

    def step():
        return nacho_amd.gpu_clip_grad_norm(tensors, 1.0, out=outs)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        for t in tensors:
            t.normal_()
        graph.replay()
        torch.cuda.synchronize()
        norm, there = got.clone(), [o.clone() for o in outs]
        assert torch.equal(norm, step())
        assert all(torch.equal(a, b) for a, b in zip(there, outs))


def test_a_write_is_noticed(gpu):
    x = torch.randn(5, device=gpu, requires_grad=True)
    w = torch.randn(5, device=gpu)
    y = (x * w).sum()
    nacho_amd.gpu_clip_grad_norm([w], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals(gpu):
    a, b = torch.ones(100, device=gpu), torch.ones(10, 10, device=gpu)
    f, norm = nacho_amd.gpu_clip_grad_norm, nacho_amd.gpu_grad_norm
    for call, error, text in [
            (lambda: norm([]), ValueError, "at least one"),
            (lambda: norm([None]), ValueError, "at least one"),
            (lambda: norm([a, 3.0]), TypeError, "expected a torch.Tensor"),
            (lambda: norm([a, b.cpu()]), ValueError, "GPU tensor"),
            (lambda: norm([a, b.double()]), TypeError, r"tensors\[1\]: expected dtype"),
            (lambda: norm([a.to_sparse()]), TypeError, "strided"),
            (lambda: f([a], -1.0), ValueError, "max_norm"),
            (lambda: f([a], math.nan), ValueError, "max_norm"),
            (lambda: f([a], 1e39), ValueError, "max_norm"),
            (lambda: f([a, torch.ones(3, device=gpu, requires_grad=True)], 1.0), ValueError,
             "not the parameters"),
            (lambda: f([a], 1.0, out=[a.clone().requires_grad_()]), ValueError,
             "not the parameters"),
            (lambda: f([a, a], 1.0), ValueError, "share memory"),
            (lambda: f([a, a[3:7]], 1.0), ValueError, "share memory"),
            (lambda: f([a[:90], b], 1.0, out=[a[10:], b]), ValueError, "share memory"),
            (lambda: f([a, b], 1.0, out=[b.view(-1), a.view(10, 10)]), ValueError, "share memory"),
            (lambda: f([b[:, 2:5]], 1.0), ValueError, "next to each other"),
            (lambda: f([a[:1].expand(5)], 1.0), ValueError, "next to each other"),
            (lambda: f([a], 1.0, out=[b]), ValueError, "shape"),
            (lambda: f([a], 1.0, out=[]), ValueError, "tensor for each"),
            (lambda: f([a], 1.0, out=[None]), ValueError, "tensor for each"),
            (lambda: f([a], 1.0, out=[a.half()]), TypeError, "expected dtype"),
            (lambda: f([b], 1.0, out=[torch.ones(10, 20, device=gpu)[:, ::2]]), ValueError,
             "next to each other")]:
        with pytest.raises(error, match=text):
            call()
    assert (a == 1).all() and (b == 1).all()
    f([a, b], 1.0, out=[a.clone(), b.clone()])
    both = [a, a]  # read twice, written apart
    assert abs(float(f(both, 1.0, out=[a.clone(), a.clone()])) - math.sqrt(200)) < 1e-5


def test_a_norm_has_no_gradient(gpu):
    """What would lose its gradient or its tangent without a word raises."""
    a, b = torch.randn(50, device=gpu, requires_grad=True), torch.randn(7, 3, device=gpu)
    norm = nacho_amd.gpu_grad_norm([None, 2.0 * a, b])
    assert torch.equal(norm.detach(), nacho_amd.gpu_grad_norm([2.0 * a.detach(), b]))
    with pytest.raises(RuntimeError, match="gpu_grad_norm has no gradient"):
        (a.sum() + norm).backward()
    with torch.no_grad():
        assert not nacho_amd.gpu_grad_norm(a).requires_grad
    assert not nacho_amd.gpu_grad_norm(a.detach()).requires_grad
    with pytest.raises(TypeError, match=r"tensors\[2\]: expected dtype"):
        nacho_amd.gpu_grad_norm([None, a, b.double()])


def test_refuses_tangents(gpu):
    from torch.autograd import forward_ad

    a, b = torch.randn(50, device=gpu), torch.randn(7, 3, device=gpu)
    want, before = nacho_amd.gpu_grad_norm([a, b]), b.clone()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(b, torch.ones_like(b))
        with pytest.raises(NotImplementedError, match="jvp"):
            nacho_amd.gpu_grad_norm([a, dual])
        with pytest.raises(NotImplementedError, match="jvp"):
            nacho_amd.gpu_clip_grad_norm([a, dual], 0.1)
        with pytest.raises(NotImplementedError, match="jvp"):
            nacho_amd.gpu_clip_grad_norm([b], 0.1, out=[dual])
        assert torch.equal(b, before)
        assert torch.equal(nacho_amd.gpu_grad_norm([a, b]), want)
        assert torch.equal(nacho_amd.gpu_clip_grad_norm([a, None, b], 0.1), want)
    with pytest.raises(TypeError, match="expected a torch.Tensor"):
        nacho_amd.gpu_clip_grad_norm([a, 3.0], 0.1)
