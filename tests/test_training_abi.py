"""The C entry points of a training step's ends: descriptor layouts, and refusals that come before any
HIP call.  Runs on the CPU."""

import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from tests.loss_reference import Loss, near

REPO = Path(__file__).resolve().parent.parent
P = ctypes.c_void_p
OK, INVALID, OVERFLOW = 0, -1, -2
X, Y, Z = P(0x10000), P(0x20000), P(0x30000)


@pytest.fixture(scope="module")
def lib():
    from nacho_amd import _lib

    return _lib.load()


def test_layouts_match_the_c_compiler(tmp_path):
    from nacho_amd import _lib

    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "nacho_hip.h"',
             'int main(void) { printf("sizeof %zu\\n", sizeof(nacho_gradient));']
    for field, _ in _lib.Gradient._fields_:
        lines.append(f'printf("{field} %zu\\n", offsetof(nacho_gradient, {field}));')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run([gcc, f"-I{REPO / 'include'}", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True,
                               text=True).stdout.splitlines():
        field, value = line.split()
        got = ctypes.sizeof(_lib.Gradient) if field == "sizeof" else \
            getattr(_lib.Gradient, field).offset
        assert got == int(value), field


def test_embedding_refuses(lib):
    f, b = lib.nacho_embedding, lib.nacho_embedding_backward
    good = [2, 10, 100, 64, 1.0, X, 8, Y, 64, Z, None]
    for at, bad, want in ((0, 3, INVALID), (0, -1, INVALID), (1, -1, INVALID), (2, -1, INVALID),
                          (3, -1, INVALID), (4, math.nan, INVALID), (4, math.inf, INVALID),
                          (5, None, INVALID), (5, P(0x10004), INVALID), (6, 2, INVALID),
                          (7, None, INVALID), (7, P(0x20001), INVALID), (9, None, INVALID),
                          (9, P(0x30001), INVALID), (2, (1 << 30) + 1, OVERFLOW),
                          (1, 1 << 31, OVERFLOW)):
        args = list(good)
        args[at] = bad
        assert f(*args) == want, (at, bad)
        assert b(*args, None) == want, (at, bad)
    assert f(2, 0, 100, 64, 1.0, None, 8, Y, 64, None, None) == OK
    assert f(2, 10, 100, 0, 1.0, X, 8, Y, 0, None, None) == OK
    assert b(2, 10, 0, 64, 1.0, X, 8, Y, 64, None, None, None) == OK
    assert b(0, 1 << 30, 100, 1 << 12, 1.0, X, 8, Y, 1 << 12, Z, None, None) == OVERFLOW


def test_loss_refuses(lib):
    f, b = lib.nacho_linear_cross_entropy, lib.nacho_linear_cross_entropy_backward
    good = [2, 10, 100, 64, 1.0, 1, X, 64, Y, 64, Z, 8]
    for at, bad, want in ((0, 3, INVALID), (1, -1, INVALID), (2, 0, INVALID), (3, 0, INVALID),
                          (4, math.nan, INVALID), (5, 3, INVALID), (5, -1, INVALID),
                          (6, None, INVALID), (6, P(0x10001), INVALID), (8, None, INVALID),
                          (8, P(0x20001), INVALID), (9, 63, INVALID), (10, None, INVALID),
                          (10, P(0x30004), INVALID), (11, 2, INVALID),
                          (1, (1 << 30) + 1, OVERFLOW), (2, (1 << 30) + 1, OVERFLOW),
                          (3, (1 << 20) + 1, OVERFLOW)):
        args = list(good)
        args[at] = bad
        if at == 3:
            args[7] = args[9] = 1 << 21
        assert f(*args, X, Y, None, None) == want, (at, bad)
        assert b(*args, X, Y, Z, Z, None, None) == want, (at, bad)
    assert f(*good, None, None, None, None) == INVALID
    assert b(*good, None, Y, Z, Z, None, None) == INVALID
    assert b(*good, X, None, Z, Z, None, None) == INVALID
    assert b(*good, X, Y, P(0x30001), Z, None, None) == INVALID
    assert b(*good, X, Y, None, None, None, None) == OK
    none = list(good)
    none[1], none[5] = 0, 0
    assert f(*none, None, None, None, None) == OK
    assert b(*none, None, None, Z, None, None, None) == OK


def test_clip_refuses(lib):
    from nacho_amd import _lib

    def one(**changes):
        t = _lib.Gradient(0x10000, 0x20000, 100, 2, 2)
        for name, value in changes.items():
            setattr(t, name, value)
        return ctypes.byref(t)

    clip, norm = lib.nacho_clip_grad_norm, lib.nacho_grad_norm
    for changes in (dict(size=-1), dict(dtype=3), dict(dtype=-1), dict(data=None),
                    dict(data=0x10001)):
        assert norm(one(**changes), 1, X, None, None) == INVALID, changes
        assert clip(one(**changes), 1, 1.0, X, None, None) == INVALID, changes
    for changes in (dict(out=None), dict(out=0x20001), dict(out_dtype=1), dict(out_dtype=5)):
        assert clip(one(**changes), 1, 1.0, X, None, None) == INVALID, changes
    assert clip(one(), 1, -1.0, X, None, None) == INVALID
    assert clip(one(), 1, math.nan, X, None, None) == INVALID
    assert clip(one(), -1, 1.0, X, None, None) == INVALID
    assert norm(None, 1, X, None, None) == INVALID
    assert norm(one(), 1, None, None, None) == INVALID
    assert norm(one(size=1 << 40), 1, X, None, None) == OVERFLOW


def test_clip_refuses_wider_elements_in_place(lib):
    """float32 written where 16-bit elements are still to be read, past the end of their memory."""
    from nacho_amd import _lib

    for dtype in (1, 2):
        t = _lib.Gradient(0x10000, 0x10000, 100, dtype, 0)
        assert lib.nacho_clip_grad_norm(ctypes.byref(t), 1, 1.0, X, None, None) == INVALID


def test_arguments_that_are_refused_before_the_library():
    import nacho_amd

    t = torch.zeros(3, 4)
    for call, error, text in [
            (lambda: nacho_amd.gpu_embedding(t.long(), t), ValueError, "GPU tensor"),
            (lambda: nacho_amd.gpu_embedding(None, t), TypeError, "torch.Tensor"),
            (lambda: nacho_amd.gpu_linear_cross_entropy(t, t, t.long()), ValueError, "GPU tensor"),
            (lambda: nacho_amd.gpu_grad_norm([t]), ValueError, "GPU tensor"),
            (lambda: nacho_amd.gpu_grad_norm([]), ValueError, "at least one"),
            (lambda: nacho_amd.gpu_clip_grad_norm([t], 1.0), ValueError, "GPU tensor")]:
        with pytest.raises(error, match=text):
            call()


# ---- the reference of the GPU tests ---------------------------------------------------

@pytest.mark.parametrize("reduction", ("none", "mean", "sum"))
def test_reference_is_autograds(reduction):
    g = torch.Generator().manual_seed(0)
    x, table = torch.randn(40, 16, generator=g), torch.randn(30, 16, generator=g)
    targets = torch.randint(-3, 33, (40,), generator=g)
    dloss = torch.rand(40, generator=g) if reduction == "none" else torch.tensor(0.7)
    want = Loss(x, table, targets, 0.5, reduction, dloss)
    ops = [t.double().requires_grad_() for t in (x, table)]
    kept = torch.where((targets >= 0) & (targets < 30), targets, -100)
    loss = torch.nn.functional.cross_entropy(0.5 * ops[0] @ ops[1].T, kept, reduction=reduction)
    grads = torch.autograd.grad(loss, ops, dloss.double())
    for got, name in zip((loss, *grads), ("loss", "dx", "dtable")):
        assert torch.allclose(got.detach(), getattr(want, name), rtol=0, atol=1e-12), name


def test_the_comparison_sees_a_mistake():
    """A word too few, another scale, a neighbour's target, a gradient without its factor."""
    g = torch.Generator().manual_seed(1)
    x, table = torch.randn(40, 32, generator=g), torch.randn(50, 32, generator=g)
    targets = torch.randint(0, 40, (40,), generator=g)
    dloss = torch.tensor(0.7)
    want = Loss(x, table, targets, 1.0, "mean", dloss)
    for other, names in ((Loss(x, table[:49], targets, 1.0, "mean", dloss), ("loss", "dx")),
                         (Loss(x, table, targets, 1.001, "mean", dloss), ("loss", "dx", "dtable")),
                         (Loss(x, table, targets + 1, 1.0, "mean", dloss), ("loss", "dx", "dtable")),
                         (Loss(x, table, targets, 1.0, "sum", dloss), ("loss", "dx", "dtable"))):
        for name in names:
            with pytest.raises(AssertionError):
                near(getattr(other, name).float(), getattr(want, name), getattr(want, name + "_off"))
