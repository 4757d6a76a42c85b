"""Block means, scores, selection and block attention with its gradients against their
definitions in float64, at the sizes, masks and layouts where they can go wrong."""

import math

import pytest
import torch

import nacho_amd
from tests import block_reference as ref

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _ids(g, batch, queries, kv_heads, keys, block, count):
    """Ids around the query's reach, unsorted: some repeated, some past the end, some -1."""
    n = (keys + block - 1) // block
    shape = (batch, queries, kv_heads, count)
    ids = torch.randint(-1, n + 1, shape, generator=g, dtype=torch.int32)
    if count:
        place = keys - queries + torch.arange(queries)
        own = (place.clamp(min=0) // block).int()[None, :, None].expand(shape[:3])
        ids[..., 0] = torch.where(torch.rand(shape[:3], generator=g) < 0.8, own, ids[..., 0])
    return ids


def _operands(seed, dtype, batch, queries, keys, q_heads, kv_heads, dim, block, count):
    g = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    return (normal(batch, queries, q_heads, dim), normal(batch, keys, kv_heads, dim),
            normal(batch, keys, kv_heads, dim),
            _ids(g, batch, queries, kv_heads, keys, block, count),
            normal(batch, queries, q_heads, dim))


def _check(gpu, q, k, v, ids, dout, block, lengths=None, causal=True, scale=None):
    want = ref.Attention(q, k, v, ids, block, lengths, causal, scale, dout)
    dev = [x.to(gpu) for x in (q, k, v)]
    for x in dev:
        x.requires_grad_()
    len_dev = None if lengths is None else lengths.to(gpu)
    how = dict(lengths=len_dev, causal=causal, scale=scale)
    out, lse = nacho_amd.gpu_block_attention(*dev, ids.to(gpu), block, return_lse=True, **how)
    ref.near(out, want.out, want.out_off, "out")
    ref.near(lse, want.lse, want.lse_off, "lse")
    grads = torch.autograd.grad(out, dev, dout.to(gpu))
    for got, name in zip(grads, ("dq", "dk", "dv")):
        ref.near(got, getattr(want, name), getattr(want, name + "_off"), name)
    with torch.no_grad():
        again = nacho_amd.gpu_block_attention(*dev, ids.to(gpu), block, **how)
    assert torch.equal(again, out)
    return out, grads


# batch, queries, keys, q_heads, kv_heads, dim, block, count.  Fewer than 256 tiles of 64 rows
# take the kernel for few rows, more the one for many.
FEW = [
    (1, 1, 1, 1, 1, 8, 32, 1),
    (2, 1, 333, 4, 4, 64, 32, 5),
    (1, 1, 2100, 8, 2, 128, 64, 9),
    (3, 2, 130, 6, 2, 80, 64, 2),
    (1, 3, 700, 20, 1, 40, 128, 4),     # a group larger than the tile of 16 rows
    (1, 5, 64, 70, 1, 24, 32, 1),       # and than the one of 64
    (2, 65, 65, 3, 3, 96, 32, 3),
    (1, 200, 257, 5, 5, 128, 128, 2),
    (1, 129, 1024, 15, 3, 72, 64, 6),
]
MANY = [
    (2, 300, 300, 32, 8, 64, 64, 3),
    (1, 1100, 1133, 16, 16, 128, 64, 7),
    (3, 333, 400, 21, 7, 80, 32, 6),
    (4, 129, 129, 128, 2, 16, 32, 2),   # a group as large as the tile
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes", FEW, ids=str)
def test_few_rows(gpu, sizes, dtype):
    _check(gpu, *_operands(1, dtype, *sizes), sizes[6])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes", MANY, ids=str)
def test_many_rows(gpu, sizes, dtype):
    _check(gpu, *_operands(2, dtype, *sizes), sizes[6])


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("sizes", [FEW[3], FEW[8], MANY[0]], ids=str)
def test_ragged_lengths(gpu, sizes, causal):
    """Lengths from 0 to all keys, some shorter than the queries; what lies past a length is
    never used, whatever it holds."""
    q, k, v, ids, dout = _operands(3, torch.bfloat16, *sizes)
    batch, keys = k.shape[:2]
    for first in (0, 1, 31, keys // 2, keys - 1):
        lengths = torch.tensor([first, keys, max(1, keys - 70)][:batch], dtype=torch.int32)
        k2, v2 = k.clone(), v.clone()
        for b in range(batch):
            k2[b, int(lengths[b]):] = float("nan")
            v2[b, int(lengths[b]):] = float("inf")
        _check(gpu, q, k2, v2, ids, dout, sizes[6], lengths, causal)


def test_lengths_past_the_cache_are_its_end(gpu):
    q, k, v, ids, _ = _operands(4, torch.float16, *FEW[1])
    far = torch.tensor([10 ** 6, -5], dtype=torch.int32)
    near = torch.tensor([k.shape[1], 0], dtype=torch.int32)
    got = [nacho_amd.gpu_block_attention(q.to(gpu), k.to(gpu), v.to(gpu), ids.to(gpu), 32,
                                         lengths=x.to(gpu)) for x in (far, near)]
    assert torch.equal(*got) and not got[0][1].any()


@pytest.mark.parametrize("sizes", [FEW[1], MANY[0]], ids=str)
def test_rows_without_blocks(gpu, sizes):
    """Every row, and then every other row, selects nothing: zeros, -inf and no gradient."""
    q, k, v, ids, dout = _operands(5, torch.float32, *sizes)
    ids[:, ::2] = -1
    _check(gpu, q, k, v, ids, dout, sizes[6])
    out, grads = _check(gpu, q, k, v, torch.full_like(ids, -1), dout, sizes[6])
    assert not out.any() and not any(x.any() for x in grads)
    _check(gpu, q, k, v, ids[..., :0], dout, sizes[6])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes", [(2, 300, 300, 32, 8, 64, 64, 2), (1, 64, 200, 4, 2, 128, 32, 2),
                                   (1, 3, 200, 4, 2, 72, 64, 1), (2, 1, 200, 4, 2, 72, 64, 2)],
                         ids=str)
def test_not_finite_in_masked_places(gpu, sizes, dtype):
    """Keys and values that are not finite reach the queries that see them, and no others: not
    those that other queries of their tile selected, nor later keys of a query's own block."""
    q, k, v, ids, dout = _operands(17, dtype, *sizes)
    block, (batch, keys, kv_heads, dim) = sizes[6], k.shape
    group = q.shape[2] // kv_heads
    bad_k, bad_v = k.clone(), v.clone()
    for b in range(batch):
        for h in range(kv_heads):
            bad_v[b, keys - 40 + h, h, 3] = math.inf
            bad_v[b, 17 + h, h, dim - 1] = math.nan
            bad_k[b, keys - 1, h] = math.nan  # seen by the last query alone
            bad_k[b, keys // 2, h, 1] = -math.inf
    hurt = ~(torch.isfinite(bad_k).all(-1) & torch.isfinite(bad_v).all(-1))  # [b, keys, h]
    see = ref.visible(ids, q.shape[1], keys, block, None, True)
    sees = (see & hurt.transpose(1, 2)[:, :, None]).any(-1).transpose(1, 2)  # [b, queries, h]
    sees = sees.repeat_interleave(group, -1)
    assert sizes[1] == 1 or (sees.any() and not sees.all())
    sees_v = torch.stack([(see & ~torch.isfinite(bad_v[..., c]).transpose(1, 2)[:, :, None])
                          .any(-1).transpose(1, 2) for c in range(dim)], -1)
    sees_v = sees_v.repeat_interleave(group, 2)
    sees_k = (see & ~torch.isfinite(bad_k).all(-1).transpose(1, 2)[:, :, None]).any(-1)
    sees_k = sees_k.transpose(1, 2).repeat_interleave(group, -1)

    good = torch.nan_to_num(bad_k, 0.0, 0.0, 0.0), torch.nan_to_num(bad_v, 0.0, 0.0, 0.0)
    want = ref.Attention(q, *good, ids, block, dout=dout)
    dev = [x.to(gpu).requires_grad_() for x in (q, bad_k, bad_v)]
    out, lse = nacho_amd.gpu_block_attention(*dev, ids.to(gpu), block, return_lse=True)
    dq, = torch.autograd.grad(out, dev[:1], dout.to(gpu))
    out, lse, dq = out.detach().cpu(), lse.cpu(), dq.cpu()
    clean = ~sees_k[..., None] & ~sees_v
    none = torch.zeros((), dtype=torch.float64)

    def check(got, name, where):
        ref.near(torch.where(where, got.double(), none),
                 torch.where(where, getattr(want, name), none),
                 getattr(want, name + "_off"), name)

    check(out, "out", clean)
    check(lse, "lse", ~sees_k)
    check(dq, "dq", ~sees[..., None].expand_as(dq))
    assert not torch.isfinite(out[sees_v & ~sees_k[..., None]]).any()


@pytest.mark.parametrize("batch,queries,keys", [(0, 4, 40), (2, 0, 40), (2, 4, 0)])
def test_empty_operands(gpu, batch, queries, keys):
    q, k, v, _, dout = _operands(6, torch.bfloat16, batch, queries, keys, 4, 2, 32, 32, 1)
    ids = torch.zeros(batch, queries, 2, 1, dtype=torch.int32)
    dev = [x.to(gpu).requires_grad_() for x in (q, k, v)]
    out = nacho_amd.gpu_block_attention(*dev, ids.to(gpu), 32)
    grads = torch.autograd.grad(out, dev, dout.to(gpu))
    assert out.shape == q.shape and not out.any()
    for x, y in zip(dev, grads):
        assert x.shape == y.shape and not y.any()


@pytest.mark.parametrize("scale", (0.0, -0.3, 2.5))
def test_scales(gpu, scale):
    _check(gpu, *_operands(7, torch.float32, *FEW[6]), 32, scale=scale)


def test_large_logits(gpu):
    """Scores in the thousands: the running maximum keeps every exponential in range."""
    q, k, v, ids, dout = _operands(8, torch.float32, *FEW[6])
    _check(gpu, 60 * q, 60 * k, v, ids, dout, 32)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layouts(gpu, dtype):
    """Head-major tensors, slices of larger ones, and rows that no 16-byte piece starts: all
    give what their contiguous copies give."""
    q, k, v, ids, dout = (x.to(gpu) for x in _operands(9, dtype, *FEW[4]))
    want = nacho_amd.gpu_block_attention(q, k, v, ids, 128)

    def head_major(x):
        return x.transpose(1, 2).contiguous().transpose(1, 2)

    def sliced(x, by):
        b, r, h, d = x.shape
        big = torch.full((b, r + 2, h + 1, d + by), float("nan"), dtype=x.dtype, device=gpu)
        view = big[:, 1:-1, 1:, by // 2:by // 2 + d]
        view.copy_(x)
        return view

    def columns(x):
        return x.permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0)

    for make in (head_major, lambda x: sliced(x, 16), lambda x: sliced(x, 6), columns):
        ops = [make(x).requires_grad_() for x in (q, k, v)]
        out = nacho_amd.gpu_block_attention(*ops, ids, 128)
        assert torch.equal(out, want)
        grads = torch.autograd.grad(out, ops, make(dout))
        base = [x.clone().requires_grad_() for x in (q, k, v)]
        same = torch.autograd.grad(nacho_amd.gpu_block_attention(*base, ids, 128), base, dout)
        assert all(torch.equal(x, y) for x, y in zip(grads, same))


def test_broadcast_gradient(gpu):
    """An output summed: its gradient is one number with strides of 0."""
    q, k, v, ids, dout = _operands(10, torch.float32, *FEW[6])
    dev = [x.to(gpu).requires_grad_() for x in (q, k, v)]
    nacho_amd.gpu_block_attention(*dev, ids.to(gpu), 32).sum().backward()
    want = ref.Attention(q, k, v, ids, 32, dout=torch.ones_like(dout))
    for x, name in zip(dev, ("dq", "dk", "dv")):
        ref.near(x.grad, getattr(want, name), getattr(want, name + "_off"), name)


def test_gradient_against_differences(gpu):
    """The gradients of q, k and v along random directions, against central differences of the
    float64 definition."""
    q, k, v, ids, dout = _operands(11, torch.float32, *FEW[8])
    dev = [x.to(gpu).requires_grad_() for x in (q, k, v)]
    out = nacho_amd.gpu_block_attention(*dev, ids.to(gpu), 64)
    grads = torch.autograd.grad(out, dev, dout.to(gpu))
    g = torch.Generator().manual_seed(1)
    want = ref.Attention(q, k, v, ids, 64, dout=dout)
    # (the definition takes its roundoff from the type that is written here)
    ref.ROUNDOFF[torch.float64] = ref.TINY[torch.float64] = 0.0
    try:
        for i, name in enumerate(("dq", "dk", "dv")):
            step = torch.randn(dev[i].shape, generator=g, dtype=torch.float64)
            h = 1e-5
            sides = []
            for sign in (1.0, -1.0):
                ops = [x.double() for x in (q, k, v)]
                ops[i] = ops[i] + sign * h * step
                sides.append((ref.Attention(*ops, ids, 64).out * dout.double()).sum())
            slope = float(sides[0] - sides[1]) / (2 * h)
            got = float((grads[i].double().cpu() * step).sum())
            off = float((getattr(want, name + "_off") * step.abs()).sum())
            # the differences' own error is of the order h^2 of the third derivative
            assert abs(got - slope) <= off + 1e-6 * (1.0 + abs(slope)), name
    finally:
        del ref.ROUNDOFF[torch.float64], ref.TINY[torch.float64]


def test_long_cache_offsets(gpu):
    """Rows of a cache past 2^31 elements from its start."""
    keys, heads, dim, block = 140, 2, 64, 32
    stride = (1 << 24) + 8  # 140 rows of it: 2.35e9 elements
    flat = torch.zeros(stride * (keys - 1) + heads * dim, dtype=torch.bfloat16, device=gpu)
    cache = flat.as_strided((1, keys, heads, dim), (0, stride, dim, 1))
    q, k, v, ids, dout = _operands(12, torch.bfloat16, 1, 3, keys, 4, heads, dim, block, 5)
    cache.copy_(k.to(gpu))
    want = ref.Attention(q, k, v, ids, block, dout=dout)
    ops = [q.to(gpu).requires_grad_(), cache, v.to(gpu).requires_grad_()]
    out = nacho_amd.gpu_block_attention(*ops, ids.to(gpu), block)
    ref.near(out, want.out, want.out_off, "out")
    dq, dv = torch.autograd.grad(out, (ops[0], ops[2]), dout.to(gpu))
    ref.near(dq, want.dq, want.dq_off, "dq")
    ref.near(dv, want.dv, want.dv_off, "dv")
    mean, off = ref.means(k, block)
    ref.near(nacho_amd.gpu_block_means(cache, block), mean, off, "means")


def test_many_blocks(gpu):
    """More blocks than one window of the lists holds (512), a token in each window."""
    keys, block = 32 * 1500 + 7, 32
    g = torch.Generator().manual_seed(13)
    q = torch.randn(1, 2, 4, 32, generator=g)
    k, v = torch.randn(2, 1, keys, 2, 32, generator=g)
    ids = torch.tensor([0, 511, 512, 513, 1023, 1024, 1499, 1500], dtype=torch.int32)
    ids = ids.expand(1, 2, 2, 8).contiguous()
    _check(gpu, q, k, v, ids, torch.ones_like(q), block)


def test_another_stream(gpu):
    q, k, v, ids, dout = _operands(14, torch.float16, *MANY[0])
    want = ref.Attention(q, k, v, ids, 64)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = nacho_amd.gpu_block_attention(q.to(gpu), k.to(gpu), v.to(gpu), ids.to(gpu), 64)
    torch.cuda.current_stream().wait_stream(side)
    ref.near(out, want.out, want.out_off, "out")


def test_graph_replays(gpu):
    """One decoding step, scored, selected and attended, recorded once: each replay gives the
    eager result for the operands that are there then."""
    q, k, v, _, _ = (x.to(gpu) for x in _operands(15, torch.bfloat16, 2, 1, 900, 8, 2, 64, 32, 1))
    lengths = torch.tensor([900, 411], dtype=torch.int32, device=gpu)

    def step():
        means = nacho_amd.gpu_block_means(k, 32, lengths)
        scores = nacho_amd.gpu_block_scores(q, means, 32, 900, lengths)
        ids = nacho_amd.gpu_block_select(scores, 6, 32, 900, lengths)
        return ids, nacho_amd.gpu_block_attention(q, k, v, ids, 32, lengths)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        q.normal_()
        lengths.copy_(torch.tensor([900 - 13 * i, 411 + 40 * i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, step()):
            assert torch.equal(x, y)


# ---- means, scores, selection ---------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes", [(1, 1, 1, 8, 32), (2, 333, 3, 80, 32), (3, 640, 2, 128, 64),
                                   (1, 300, 5, 64, 128)], ids=str)
def test_means(gpu, sizes, dtype):
    batch, keys, heads, dim, block = sizes
    g = torch.Generator().manual_seed(20)
    k = torch.randn(batch, keys, heads, dim, generator=g).to(dtype)
    for lengths in (None, torch.tensor([0, keys, keys // 2][:batch], dtype=torch.int32)):
        want, off = ref.means(k, block, lengths)
        filled = k.clone()
        if lengths is not None:
            for b in range(batch):
                filled[b, int(lengths[b]):] = float("nan")
        got = nacho_amd.gpu_block_means(filled.to(gpu), block,
                                        None if lengths is None else lengths.to(gpu))
        ref.near(got, want, off, "means")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("sizes", [(1, 1, 1, 1, 1, 8, 32), (2, 70, 333, 6, 2, 80, 32),
                                   (3, 1, 9000, 20, 4, 128, 64), (2, 130, 64, 7, 7, 40, 128)],
                         ids=str)
def test_scores(gpu, sizes, causal, dtype):
    batch, queries, keys, q_heads, kv_heads, dim, block = sizes
    g = torch.Generator().manual_seed(21)
    q = torch.randn(batch, queries, q_heads, dim, generator=g).to(dtype)
    mean = torch.randn(batch, (keys + block - 1) // block, kv_heads, dim, generator=g)
    for lengths in (None, torch.tensor([keys // 3, 0, keys][:batch], dtype=torch.int32)):
        want, off = ref.scores(q, mean, block, keys, lengths, causal)
        got = nacho_amd.gpu_block_scores(q.to(gpu), mean.to(gpu), block, keys, causal=causal,
                                         lengths=None if lengths is None else lengths.to(gpu))
        ref.near(got, want, off, "scores")


@pytest.mark.parametrize("sizes", [(1, 1, 1, 1, 32, 3), (2, 70, 2, 333, 32, 4),
                                   (2, 3, 2, 64 * 300, 64, 17), (1, 2, 1, 32 * 1900, 32, 100),
                                   (1, 2, 2, 32 * 2500, 32, 9), (1, 40, 1, 32, 32, 2)], ids=str)
@pytest.mark.parametrize("kind", ("normal", "ties", "holes"))
def test_select(gpu, sizes, kind):
    """Equal scores go to the lowest id; -inf and NaN are no candidates; 0 and -0 are equal."""
    batch, queries, heads, keys, block, count = sizes
    g = torch.Generator().manual_seed(22)
    n = (keys + block - 1) // block
    s = torch.randn(batch, queries, heads, n, generator=g)
    if kind == "ties":
        s = (s * 2).round() / 2 * torch.where(torch.rand(s.shape, generator=g) < 0.5, 1.0, -1.0)
    if kind == "holes":
        u = torch.rand(s.shape, generator=g)
        s[u < 0.3], s[u > 0.7] = -math.inf, math.nan
        s[(u > 0.5) & (u < 0.55)] = math.inf
        s[(u > 0.6) & (u < 0.65)] = torch.finfo(torch.float32).min
    for lengths in (None, torch.tensor([keys // 2, 0][:batch], dtype=torch.int32)):
        for causal, sink, local in ((True, 1, 1), (True, 0, 0), (False, 2, 3), (True, 3, 50)):
            want = ref.select(s, count, block, keys, lengths, causal, sink, local)
            got = nacho_amd.gpu_block_select(
                s.to(gpu), count, block, keys, None if lengths is None else lengths.to(gpu),
                causal, sink, local)
            assert torch.equal(got.cpu(), want), (causal, sink, local)


# ---- refusals -------------------------------------------------------------------------

def test_refusals(gpu):
    q, k, v, ids, dout = (x.to(gpu) for x in _operands(16, torch.bfloat16, *FEW[3]))
    f = nacho_amd.gpu_block_attention
    bad = [
        ((q.cpu(), k, v, ids, 64), ValueError, "GPU tensor"),
        ((q, k.cpu(), v, ids, 64), ValueError, "GPU tensor"),
        ((q, k.float(), v, ids, 64), TypeError, "k: expected dtype"),
        ((q.double(), k, v, ids, 64), TypeError, "q: expected dtype"),
        ((q, k, v[:, 1:], ids, 64), ValueError, "do not fit"),
        ((q, k, v, ids.long(), 64), TypeError, "blocks"),
        ((q, k, v, ids[:, 1:], 64), ValueError, "blocks"),
        ((q, k, v, ids, 48), ValueError, "block must be"),
        ((q[:, :, :5], k, v, ids, 64), ValueError, "multiple"),
        ((q[..., :12], k[..., :12], v[..., :12], ids, 64), ValueError, "head_dim"),
        ((q[0], k, v, ids, 64), ValueError, "dimensions"),
        ((q, k, v, None, 64), TypeError, "blocks"),
    ]
    for args, error, text in bad:
        with pytest.raises(error, match=text):
            f(*args)
    with pytest.raises(ValueError, match="lengths"):
        f(q, k, v, ids, 64, lengths=torch.zeros(2, dtype=torch.int32, device=gpu))
    with pytest.raises(TypeError, match="lengths"):
        f(q, k, v, ids, 64, lengths=torch.zeros(3, device=gpu))
    with pytest.raises(ValueError, match="scale"):
        f(q, k, v, ids, 64, scale=math.inf)
    out, lse = f(q, k, v, ids, 64, return_lse=True)
    with pytest.raises(ValueError, match="lse"):
        nacho_amd.gpu_block_attention_backward(dout, q, k, v, ids, 64, out, lse[:, 1:])
    with pytest.raises(TypeError, match="dout"):
        nacho_amd.gpu_block_attention_backward(dout.float(), q, k, v, ids, 64, out, lse)
    with pytest.raises(ValueError, match="means"):
        nacho_amd.gpu_block_scores(q, nacho_amd.gpu_block_means(k, 64), 32, k.shape[1])
    with pytest.raises(ValueError, match="blocks"):
        nacho_amd.gpu_block_select(torch.zeros(1, 1, 1, 3, device=gpu), 2, 32, 32)
    with pytest.raises(ValueError, match="count"):
        nacho_amd.gpu_block_select(torch.zeros(1, 1, 1, 1, device=gpu), -2, 32, 32)


# 1024 tiles of 128 rows: a wavefront has two column tiles (heads of more than 64, 16 bits).
WIDE = [(8, 70, 200, 128, 64, 128, 64, 2), (8, 65, 140, 128, 64, 96, 32, 3)]


@pytest.mark.parametrize("dtype", TYPES[1:], ids=str)
@pytest.mark.parametrize("sizes", WIDE, ids=str)
def test_two_column_tiles(gpu, sizes, dtype):
    _check(gpu, *_operands(21, dtype, *sizes), sizes[6])


def test_two_column_tiles_of_ragged_lengths(gpu):
    q, k, v, ids, dout = _operands(22, torch.bfloat16, *WIDE[0])
    ids[:, ::3] = -1
    lengths = torch.tensor([0, 1, 69, 70, 71, 128, 199, 200], dtype=torch.int32)
    for b, length in enumerate(lengths.tolist()):
        k[b, length:], v[b, length:] = float("nan"), float("inf")
    _check(gpu, q, k, v, ids, dout, 64, lengths)


def test_two_column_tiles_and_not_finite_values(gpu):
    test_not_finite_in_masked_places(gpu, (16, 40, 200, 128, 32, 72, 64, 2), torch.bfloat16)


@pytest.mark.parametrize("blocks", (3, 64, 65, 129, 256, 300, 513, 1030, 2048, 2060))
def test_select_of_any_width(gpu, blocks):
    """A row's scores are held in 1 to 32 registers of a wavefront, or read again: every form."""
    g = torch.Generator().manual_seed(blocks)
    keys, count = 32 * blocks - 5, 40
    score = torch.randn(2, 3, 2, blocks, generator=g)
    score[1] = (score[1] * 2).round()  # many equal ones
    score[:, 1, :, ::3] = -math.inf
    lengths = torch.tensor([keys, max(3, keys // 2)], dtype=torch.int32)
    want = ref.select(score, count, 32, keys, lengths)
    got = nacho_amd.gpu_block_select(score.to(gpu), count, 32, keys, lengths.to(gpu))
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes", [(1, 3, 200, 16, 1, 72, 64, 1), (2, 4, 2100, 32, 2, 128, 64, 9),
                                   (1, 2, 130, 20, 1, 64, 32, 2), (2, 4, 95, 4, 2, 64, 32, 2)],
                         ids=str)
def test_later_keys_of_the_own_block(gpu, sizes, dtype):
    """A few new tokens: the last one's key and value, which lie in the block of those before it,
    reach none of these, also where a tile of rows is the heads of one token."""
    q, k, v, ids, dout = _operands(31, dtype, *sizes)
    queries, keys, block = sizes[1], sizes[2], sizes[6]
    ids[..., 0] = (keys - 1) // block
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[:, -1], bad_v[:, -1] = math.nan, math.inf
    k[:, -1], v[:, -1] = 0.0, 0.0
    want = ref.Attention(q, k, v, ids, block, dout=dout)
    dev = [x.to(gpu).requires_grad_() for x in (q, bad_k, bad_v)]
    out, lse = nacho_amd.gpu_block_attention(*dev, ids.to(gpu), block, return_lse=True)
    dq, = torch.autograd.grad(out, dev[:1], dout.to(gpu))
    before = (torch.arange(queries) < queries - 1)[None, :, None]
    none = torch.zeros((), dtype=torch.float64)
    for got, name in ((out, "out"), (lse, "lse"), (dq, "dq")):
        where = before.expand(lse.shape) if name == "lse" else before[..., None].expand(q.shape)
        ref.near(torch.where(where, got.detach().cpu().double(), none),
                 torch.where(where, getattr(want, name), none), getattr(want, name + "_off"),
                 name)
    assert not torch.isfinite(out[:, -1]).any()
