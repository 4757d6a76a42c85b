"""Rows of a table and the table's gradient, against plain float64 sums."""

import pytest
import torch

import nacho_amd

pytestmark = pytest.mark.gpu

ROUNDOFF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E = 2.0 ** -24
TYPES = tuple(ROUNDOFF)
# tokens, words, how their words are spread: the share of one word
SIZES = [(1, 1, 0.0), (5, 3, 0.0), (31, 100, 0.0), (32, 100, 1.0), (33, 100, 1.0), (64, 7, 0.0),
         (65, 2000, 0.3), (1000, 5, 0.0), (3000, 50000, 0.5), (8192, 300, 0.1),
         (8193, 300, 0.1), (20000, 511, 0.0), (20000, 512, 0.9), (30000, 300000, 0.2),
         (100003, 1000, 0.0), (9000, 70000000, 0.0)]


def _ids(seed, tokens, words, hot, dtype=torch.int64, left=0.1):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, words, (tokens,), generator=g)
    ids[torch.rand(tokens, generator=g) < hot] = words // 2
    none = torch.rand(tokens, generator=g) < left
    bad = torch.where(torch.rand(tokens, generator=g) < 0.5, -1, words)
    return torch.where(none, bad, ids).to(dtype)


def _near(got, want, off, what):
    over = (got.detach().double().cpu() - want).abs() - 1.01 * off
    assert not torch.isnan(over).any(), what
    assert over.numel() == 0 or float(over.max()) <= 0.0, f"{what}: {float(over.max())} past"


def _check_gradient(gpu, ids, words, width, dtype, scale=1.0, make=lambda x: x):
    g = torch.Generator().manual_seed(3)
    dout = torch.randn(*ids.shape, width, generator=g).to(dtype)
    flat = ids.reshape(-1).long()
    held = (flat >= 0) & (flat < words)
    given = make(dout.to(gpu))
    got = nacho_amd.gpu_embedding_backward(given, ids.to(gpu), words, scale=scale)
    assert got.shape == (words, width) and got.dtype == dtype
    f32 = float(torch.tensor(scale, dtype=torch.float32))
    terms = dout.reshape(-1, width)[held].double()
    # (the words that occur: a table may be larger than a float64 copy of it should be)
    some, place = torch.unique(flat[held], return_inverse=True)
    want = torch.zeros(len(some), width, dtype=torch.float64).index_add_(0, place, terms)
    size = torch.zeros_like(want).index_add_(0, place, terms.abs())
    count = torch.bincount(place, minlength=len(some))[:, None]
    u, tiny = ROUNDOFF[dtype], 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    off = abs(f32) * ((count + 1) * E * size + u * want.abs()) + tiny
    _near(got[some.to(gpu)], want * f32, off, "dtable")
    there = torch.zeros(words, dtype=torch.bool, device=gpu)
    there[some.to(gpu)] = True
    assert not (got != 0).any(1)[~there].any()
    assert torch.equal(got, nacho_amd.gpu_embedding_backward(given, ids.to(gpu), words, scale=scale))


@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_gradient_sizes(gpu, sizes):
    ids = _ids(1, *sizes, dtype=torch.int32 if sizes[0] % 2 else torch.int64)
    _check_gradient(gpu, ids, sizes[1], 8 if sizes[1] > 1 << 20 else 40, torch.float32)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width", (1, 7, 8, 64, 333, 1000, 4096, 5001))
def test_gradient_widths(gpu, width, dtype):
    _check_gradient(gpu, _ids(2, 300, 90, 0.3), 90, width, dtype, scale=1.7)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width", (1, 7, 8, 64, 333, 2048, 4096, 5001))
@pytest.mark.parametrize("scale", (1.0, 45.25))
def test_rows(gpu, width, dtype, scale):
    for tokens, words, kind in ((1, 1, torch.int64), (53, 31, torch.int32), (700, 5, torch.int64)):
        ids = _ids(4, tokens, words, 0.0, kind)
        table = torch.randn(words, width, generator=torch.Generator().manual_seed(5)).to(dtype)
        got = nacho_amd.gpu_embedding(ids.to(gpu), table.to(gpu), scale=scale).cpu()
        held = (ids >= 0) & (ids < words)
        want = torch.zeros(tokens, width, dtype=dtype)
        want[held] = (table.float() * scale).to(dtype)[ids[held].long()]
        assert torch.equal(got, want)


def test_ids_of_other_shapes(gpu):
    table = torch.randn(50, 24, device=gpu, requires_grad=True)
    ids = _ids(6, 60, 50, 0.0, left=0.0).to(gpu)
    want = nacho_amd.gpu_embedding(ids, table).detach()
    for shaped in (ids.view(5, 12), ids.view(3, 4, 5)):
        got = nacho_amd.gpu_embedding(shaped, table)
        assert torch.equal(got, want.view(*shaped.shape, 24))
    got = nacho_amd.gpu_embedding(ids.view(5, 12).t(), table)
    assert torch.equal(got, want.view(5, 12, 24).transpose(0, 1))
    assert torch.equal(nacho_amd.gpu_embedding(ids[7], table), want[7])
    wide = torch.stack((ids, ids + (1 << 40)), 1)  # what is past 32 bits counts
    assert not nacho_amd.gpu_embedding(wide, table)[:, 1].any()
    big = torch.zeros(60, 3, dtype=torch.int64, device=gpu)
    big[:, 1] = ids
    assert torch.equal(nacho_amd.gpu_embedding(big[:, 1], table), want)


def test_nothing(gpu):
    table = torch.randn(50, 24, device=gpu, requires_grad=True)
    none = torch.zeros(0, 3, dtype=torch.long, device=gpu)
    out = nacho_amd.gpu_embedding(none, table)
    assert out.shape == (0, 3, 24)
    assert not torch.autograd.grad(out.sum(), table)[0].any()
    ids = torch.zeros(4, dtype=torch.long, device=gpu)
    assert not nacho_amd.gpu_embedding(ids, table[:0]).any()
    assert nacho_amd.gpu_embedding_backward(torch.ones(4, 24, device=gpu), ids, 0).shape == (0, 24)
    assert nacho_amd.gpu_embedding(ids, table[:, :0]).shape == (4, 0)
    out = nacho_amd.gpu_embedding(ids - 1, table)
    assert not out.any() and not torch.autograd.grad(out.sum(), table)[0].any()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layouts(gpu, dtype):
    """Tables and gradients that are parts of wider ones, between 16-byte pieces, and columns."""
    def sliced(by):
        def make(x):
            big = torch.full((x.shape[0] + 1, x.shape[1] + by), float("nan"), dtype=x.dtype,
                             device=x.device)
            big[1:, by // 2:by // 2 + x.shape[1]] = x
            return big[1:, by // 2:by // 2 + x.shape[1]].detach()
        return make

    ids = _ids(7, 90, 40, 0.2)
    table = torch.randn(40, 64, device=gpu).to(dtype)
    want = nacho_amd.gpu_embedding(ids.to(gpu), table)
    for make in (sliced(16), sliced(6), lambda x: x.t().contiguous().t()):
        assert torch.equal(nacho_amd.gpu_embedding(ids.to(gpu), make(table)), want)
        _check_gradient(gpu, ids, 40, 64, dtype, make=make)
    one = table[3:4].expand(40, 64)
    assert torch.equal(nacho_amd.gpu_embedding(ids.to(gpu), one)[0],
                       table[3] if 0 <= int(ids[0]) < 40 else torch.zeros_like(table[3]))


def test_broadcast_gradients(gpu):
    table = torch.randn(9, 24, device=gpu, requires_grad=True)
    ids = torch.tensor([[1, 2, 1], [4, 1, -1]], device=gpu)
    nacho_amd.gpu_embedding(ids, table, scale=2.0).sum().backward()
    want = torch.zeros(9, 24, device=gpu)
    want[1], want[2], want[4] = 6.0, 2.0, 2.0
    assert torch.equal(table.grad, want)


def test_values_that_are_not_finite(gpu):
    """They reach their own word alone, and those of tokens without a word none."""
    ids = torch.tensor([3, 5, -1, 3, 9], device=gpu)
    dout = torch.ones(5, 16, device=gpu)
    dout[2], dout[1, 4] = float("nan"), float("inf")
    got = nacho_amd.gpu_embedding_backward(dout, ids, 9)
    want = torch.zeros(9, 16, device=gpu)
    want[3], want[5] = 2.0, 1.0
    want[5, 4] = float("inf")
    assert torch.equal(got, want)
    table = torch.randn(9, 16, device=gpu)
    table[0] = float("nan")
    assert not nacho_amd.gpu_embedding(ids, table)[[2, 4]].any()


def test_graph_replays(gpu):
    for tokens, words in ((3000, 500), (20000, 1500)):
        ids = _ids(8, tokens, words, 0.2).to(gpu)
        table, dout = torch.randn(words, 64, device=gpu), torch.randn(tokens, 64, device=gpu)

        def step():
            return (nacho_amd.gpu_embedding(ids, table, scale=3.0),
                    nacho_amd.gpu_embedding_backward(dout, ids, words, scale=3.0))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for i in range(4):
            dout.normal_()
            ids.copy_(_ids(9 + i, tokens, words, 0.3 * i))
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, step()):
                assert torch.equal(a, b)


def test_autograd(gpu):
    from torch.autograd import forward_ad

    table = torch.randn(9, 24, device=gpu, requires_grad=True)
    ids = torch.tensor([1, 2, 1], device=gpu)
    out = nacho_amd.gpu_embedding(ids, table)
    ids.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    with torch.inference_mode():
        inside = ids.clone()
        assert torch.equal(nacho_amd.gpu_embedding(inside, table), table[ids])
    out = nacho_amd.gpu_embedding(inside, table)
    assert torch.equal(torch.autograd.grad(out.sum(), table)[0],
                       nacho_amd.gpu_embedding_backward(torch.ones_like(out), ids, 9))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(table.detach(), torch.ones_like(table))
        with pytest.raises(NotImplementedError, match="jvp"):
            nacho_amd.gpu_embedding(ids, dual)


def test_refusals(gpu):
    ids, table = torch.zeros(4, dtype=torch.long, device=gpu), torch.zeros(9, 8, device=gpu)
    f, b = nacho_amd.gpu_embedding, nacho_amd.gpu_embedding_backward
    dout = torch.zeros(4, 8, device=gpu)
    for call, error, text in [
            (lambda: f(ids.cpu(), table), ValueError, "ids: expected a GPU tensor"),
            (lambda: f(ids, table.cpu()), ValueError, "table: expected a GPU tensor"),
            (lambda: f(ids.float(), table), TypeError, "ids: expected dtype"),
            (lambda: f(ids, table.double()), TypeError, "table: expected dtype"),
            (lambda: f(ids, table[0]), ValueError, "table: expected 2 dimensions"),
            (lambda: f(ids, table, scale=float("inf")), ValueError, "scale"),
            (lambda: b(dout, ids, -1), ValueError, "words"),
            (lambda: b(dout, ids, (1 << 30) + 1), ValueError, "words"),
            (lambda: b(dout.double(), ids, 9), TypeError, "dout: expected dtype"),
            (lambda: b(dout[1:], ids, 9), ValueError, "dout: expected shape"),
            (lambda: b(dout, ids[None], 9), ValueError, "dout: expected shape"),
            (lambda: b(dout, ids.short(), 9), TypeError, "ids: expected dtype")]:
        with pytest.raises(error, match=text):
            call()


@pytest.mark.parametrize("tokens", (16383, 16384, 18500, 70001, 300_000))
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16), ids=str)
def test_words_of_many_runs(gpu, tokens, dtype):
    """Words that a share of a large batch has, wherever their sorted tokens begin: sums of whole numbers,
    which are exact whatever their order."""
    for width, words, hot, word in ((3, 90, 0.5, 45), (72, 7, 0.0, 0), (40, 1000, 1.0, 0),
                                    (333, 50, 0.9, 49), (1040, 3, 0.3, 1)):
        g = torch.Generator(device=gpu).manual_seed(tokens + width)
        ids = torch.randint(0, words, (tokens,), generator=g, device=gpu)
        ids[torch.rand(tokens, generator=g, device=gpu) < hot] = word
        ids[5::4001] = -1
        dout = torch.randint(-8, 9, (tokens, width), generator=g, device=gpu).to(dtype)
        got = nacho_amd.gpu_embedding_backward(dout, ids, words)
        there = (ids == torch.arange(words, device=gpu)[:, None]).float()
        assert torch.equal(got, (there @ dout.float()).to(dtype)), (width, words, hot)


def test_a_word_costs_what_the_batch_costs(gpu):
    """Half of a batch of one word takes at most twice as long as none of it."""
    tokens, words, width = 1 << 20, 32000, 64
    g = torch.Generator(device=gpu).manual_seed(1)
    dout = torch.randn(tokens, width, generator=g, device=gpu)

    def time_of(ids):
        best = float("inf")
        for _ in range(5):
            start, end = torch.cuda.Event(True), torch.cuda.Event(True)
            start.record()
            for _ in range(5):
                nacho_amd.gpu_embedding_backward(dout, ids, words)
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end))
        return best

    even = torch.randint(0, words, (tokens,), generator=g, device=gpu)
    hot = torch.where(torch.rand(tokens, generator=g, device=gpu) < 0.5, 7, even)
    time_of(even)
    assert time_of(hot) <= 2.0 * time_of(even)


@pytest.mark.parametrize("dtype,width", ((torch.float32, 257), (torch.float32, 259), (torch.float32, 515),
                                         (torch.float32, 1027), (torch.bfloat16, 513),
                                         (torch.bfloat16, 1027), (torch.bfloat16, 2051)), ids=str)
def test_words_of_many_runs_in_rows_whose_last_pieces_overlap(gpu, width, dtype):
    """A row's last piece shares columns with the one before, which is another wavefront's or workgroup's
    here: neither may read what the other has already summed."""
    tokens = 100_000
    g = torch.Generator(device=gpu).manual_seed(width)
    ids = torch.zeros(tokens, dtype=torch.int64, device=gpu)
    ids[torch.rand(tokens, generator=g, device=gpu) < 0.3] = 2
    dout = torch.randint(-8, 9, (tokens, width), generator=g, device=gpu).to(dtype)
    there = (ids == torch.arange(4, device=gpu)[:, None]).float()
    want = (there @ dout.float()).to(dtype)
    for _ in range(10):
        assert torch.equal(nacho_amd.gpu_embedding_backward(dout, ids, 4), want)
