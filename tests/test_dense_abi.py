"""The C entry points of the dense operators: descriptor layouts, and refusals that come before any
HIP call.  Runs on the CPU; also checks the references that the GPU tests compare with."""

import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from tests import block_reference as ref

REPO = Path(__file__).resolve().parent.parent
P = ctypes.c_void_p
OK, INVALID, OVERFLOW = 0, -1, -2


@pytest.fixture(scope="module")
def lib():
    from nacho_amd import _lib

    return _lib.load()


def test_layouts_match_the_c_compiler(tmp_path):
    from nacho_amd import _lib

    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    pairs = {"nacho_heads": _lib.Heads, "nacho_block_attention_args": _lib.BlockAttentionArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "nacho_hip.h"',
             "int main(void) {"]
    for name, desc in pairs.items():
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        for field, _ in desc._fields_:
            lines.append(f'printf("{name} {field} %zu\\n", offsetof({name}, {field}));')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run([gcc, f"-I{REPO / 'include'}", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True,
                               text=True).stdout.splitlines():
        name, field, value = line.split()
        desc = pairs[name]
        got = ctypes.sizeof(desc) if field == "size" else getattr(desc, field).offset
        assert got == int(value), f"{name}.{field}: ctypes {got}, C {value}"


def _args(**changes):
    from nacho_amd import _lib

    a = _lib.BlockAttentionArgs(dtype=2, batch=1, queries=4, keys=100, q_heads=4, kv_heads=2,
                                head_dim=64, block=32, count=2, causal=1, scale=0.125)
    a.blocks, a.lse = 0x1000, 0x2000
    for i, name in enumerate(("q", "k", "v", "out", "dout", "dq", "dk", "dv")):
        setattr(a, name, _lib.Heads(0x10000 * (i + 1), 1 << 20, 256, 64))
    for name, value in changes.items():
        if "." in name:
            setattr(getattr(a, name.split(".")[0]), name.split(".")[1], value)
        else:
            setattr(a, name, value)
    return a


BAD = [dict(dtype=3), dict(dtype=-1), dict(batch=-1), dict(queries=-1), dict(keys=-1),
       dict(q_heads=0), dict(kv_heads=0), dict(q_heads=5), dict(q_heads=2 * 1025),
       dict(head_dim=0), dict(head_dim=60), dict(head_dim=136), dict(block=0), dict(block=48),
       dict(block=256), dict(count=-1), dict(causal=2), dict(scale=math.inf),
       dict(scale=math.nan), dict(blocks=None), {"q.data": None}, {"k.data": None},
       {"v.data": 0x30008}, {"out.row_stride": 252}, {"k.head_stride": 4},
       {"k.row_stride": (1 << 25) + 8}, {"v.row_stride": -256}]


@pytest.mark.parametrize("changes", BAD, ids=str)
def test_attention_refuses(lib, changes):
    a = _args(**changes)
    assert lib.nacho_block_attention(ctypes.byref(a), None, None) == INVALID
    assert lib.nacho_block_attention_backward(ctypes.byref(a), None, None) == INVALID


@pytest.mark.parametrize("changes", [{"dout.data": None}, {"dq.data": 0x60004}, {"dk.data": None},
                                     {"dv.batch_stride": 4}, dict(lse=None)], ids=str)
def test_backward_refuses(lib, changes):
    a = _args(**changes)
    assert lib.nacho_block_attention_backward(ctypes.byref(a), None, None) == INVALID


def test_attention_of_nothing(lib):
    assert lib.nacho_block_attention(None, None, None) == INVALID
    assert lib.nacho_block_attention(ctypes.byref(_args(batch=0)), None, None) == OK
    a = _args(queries=0, blocks=None)
    a.q.data = a.out.data = None
    assert lib.nacho_block_attention(ctypes.byref(a), None, None) == OK
    big = _args(batch=1 << 20, queries=1 << 20)
    assert lib.nacho_block_attention(ctypes.byref(big), None, None) == OVERFLOW


def test_means_scores_select_refuse(lib):
    from nacho_amd import _lib

    h = ctypes.byref(_lib.Heads(0x10000, 1 << 20, 256, 64))
    odd = ctypes.byref(_lib.Heads(0x10004, 1 << 20, 256, 64))
    means = lib.nacho_block_means
    assert means(2, 1, 100, 2, 64, 32, None, None, P(0x1000), None) == INVALID
    assert means(2, 1, 100, 2, 64, 32, odd, None, P(0x1000), None) == INVALID
    assert means(2, 1, 100, 2, 64, 32, h, None, None, None) == INVALID
    assert means(2, 1, 100, 2, 60, 32, h, None, P(0x1000), None) == INVALID
    assert means(2, 1, 100, 2, 64, 33, h, None, P(0x1000), None) == INVALID
    assert means(2, 1, 0, 2, 64, 32, h, None, None, None) == OK
    scores = lib.nacho_block_scores
    good = (2, 1, 4, 100, 4, 2, 64, 32, 1, 0.125)
    assert scores(*good, h, None, None, P(0x1000), None) == INVALID
    assert scores(*good, h, P(0x1004), None, P(0x1000), None) == INVALID
    assert scores(*good[:9], math.nan, h, P(0x1000), None, P(0x1000), None) == INVALID
    assert scores(*good[:4], 5, *good[5:], h, P(0x1000), None, P(0x1000), None) == INVALID
    assert scores(2, 0, *good[2:], h, None, None, None, None) == OK
    select = lib.nacho_block_select
    good = (1, 4, 2, 100, 32, 3, 1, 1, 1)
    assert select(*good, None, None, P(0x1000), None) == INVALID
    assert select(*good, P(0x1000), None, None, None) == INVALID
    assert select(*good[:5], -1, *good[6:], P(0x1000), None, P(0x1000), None) == INVALID
    assert select(*good[:6], (1 << 20) + 1, 1, 1, P(0x1000), None, P(0x1000), None) == INVALID
    assert select(*good[:5], 0, *good[6:], None, None, None, None) == OK
    assert select(1 << 20, 1 << 20, *good[2:], P(0x1000), None, P(0x1000), None) == OVERFLOW


def test_routing_refuses(lib):
    x, y = P(0x1000), P(0x2000)
    route = lib.nacho_route
    assert route(x, 2, 10, 2, 4, y, y, y, None, None) == INVALID
    assert route(x, 4, -1, 2, 4, y, y, y, None, None) == INVALID
    assert route(x, 4, 10, 0, 4, y, y, y, None, None) == INVALID
    assert route(x, 4, 10, 2, 0, y, y, y, None, None) == INVALID
    assert route(x, 4, 10, 2, 2049, y, y, y, None, None) == INVALID
    assert route(None, 4, 10, 2, 4, y, y, y, None, None) == INVALID
    assert route(x, 4, 10, 2, 4, None, y, y, None, None) == INVALID
    assert route(P(0x1004), 8, 10, 2, 4, y, y, y, None, None) == INVALID
    assert route(x, 4, 1 << 31, 2, 4, y, y, y, None, None) == OVERFLOW
    dispatch = lib.nacho_dispatch
    assert dispatch(3, 10, 2, 4, 8, x, 8, y, y, x, None) == INVALID
    assert dispatch(2, 10, 2, 4, 8, None, 8, y, y, x, None) == INVALID
    assert dispatch(0, 10, 2, 4, 8, P(0x1002), 8, y, y, x, None) == INVALID
    assert dispatch(2, 0, 2, 4, 8, None, 8, None, None, None, None) == OK
    combine = lib.nacho_combine
    assert combine(2, 10, 2, -8, x, 8, None, y, x, None) == INVALID
    assert combine(2, 10, 2, 8, x, 8, None, None, x, None) == INVALID
    assert combine(2, 10, 2, 0, None, 0, None, None, None, None) == OK
    back = lib.nacho_combine_backward
    assert back(2, 10, 2, 4, 8, x, 8, None, y, y, x, 8, x, x, None) == INVALID
    assert back(2, 10, 2, 4, 8, x, 8, x, y, y, x, 8, x, None, None) == INVALID
    assert back(2, 10, 0, 4, 8, x, 8, x, y, y, x, 8, x, x, None) == INVALID


# ---- the references of the GPU tests --------------------------------------------------

@pytest.mark.parametrize("causal", (True, False))
def test_reference_gradients_are_autograds(causal):
    g = torch.Generator().manual_seed(0)
    normal = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v, dout = (normal(2, 30, 6, 16), normal(2, 50, 2, 16), normal(2, 50, 2, 16),
                     normal(2, 30, 6, 16))
    ids = torch.randint(-1, 3, (2, 30, 2, 2), generator=g, dtype=torch.int32)
    lengths = torch.tensor([50, 20])
    want = ref.Attention(q, k, v, ids, 32, lengths, causal, 0.3, dout)
    see = ref.visible(ids, 30, 50, 32, lengths, causal)[:, :, None]
    ops = [x.double().requires_grad_() for x in (q, k, v)]
    q4 = ops[0].view(2, 30, 2, 3, 16).permute(0, 2, 3, 1, 4)
    x = q4 @ ops[1].transpose(1, 2)[:, :, None].transpose(-1, -2) * 0.3
    p = torch.softmax(x.masked_fill(~see, -1e300), -1) * see
    out = (p @ ops[2].transpose(1, 2)[:, :, None]).permute(0, 3, 1, 2, 4).reshape(2, 30, 6, 16)
    grads = torch.autograd.grad((out * dout.double()).sum(), ops)
    for got, name in zip((out, *grads), ("out", "dq", "dk", "dv")):
        assert torch.allclose(got.detach(), getattr(want, name), rtol=0, atol=1e-12), name


def test_the_comparison_sees_a_mistake():
    """A key too many, a head's neighbour, an unscaled gradient: each is past its bounds."""
    g = torch.Generator().manual_seed(1)
    q, dout = torch.randn(2, 1, 40, 4, 32, generator=g)
    k, v = torch.randn(2, 1, 70, 2, 32, generator=g)
    ids = torch.randint(0, 3, (1, 40, 2, 2), generator=g, dtype=torch.int32)
    want = ref.Attention(q, k, v, ids, 32, dout=dout)
    right = ref.Attention(q, k, v, ids, 32, dout=dout)
    ref.near(right.out, want.out, want.out_off)
    wrong = [ref.Attention(q, k, v, ids, 32, causal=False, dout=dout),
             ref.Attention(q, k.flip(2), v, ids, 32, dout=dout),
             ref.Attention(q, k, v, ids, 32, scale=0.177, dout=dout)]
    for other in wrong:
        for name in ("out", "dq", "dk", "dv"):
            with pytest.raises(AssertionError):
                ref.near(getattr(other, name), getattr(want, name), getattr(want, name + "_off"))
