"""The integration guide's example of a training step's ends: its calls fit the functions' parameters,
and it runs as printed."""

import ast
import inspect
import re
from pathlib import Path

import pytest
import torch

import nacho_amd

GUIDE = Path(__file__).resolve().parent.parent / "INTEGRATION.md"


def _example():
    section = GUIDE.read_text().split("## 3c.")[1].split("\n## ")[0]
    return re.search(r"```python\n(.*?)```", section, re.S).group(1)


def test_calls_fit_the_parameters():
    calls = [n for n in ast.walk(ast.parse(_example())) if isinstance(n, ast.Call)
             and n.func.attr.startswith("gpu_")]
    assert len(calls) == 4
    for call in calls:
        named = {x.arg: None for x in call.keywords}
        inspect.signature(getattr(nacho_amd, call.func.attr)).bind(*call.args, **named)


@pytest.mark.gpu
def test_example_runs(gpu):
    table = torch.randn(50, 24, device=gpu, requires_grad=True)
    unused = torch.zeros(3, device=gpu, requires_grad=True)
    grads = [torch.randn(5, 6, device=gpu).bfloat16()]
    names = {"nacho": nacho_amd, "table": table, "parameters": [table, unused], "grads": grads,
             "ids": torch.randint(0, 50, (4, 7), device=gpu), "masters": [torch.zeros(5, 6, device=gpu)],
             "targets": torch.randint(0, 50, (4, 7), device=gpu)}
    exec(_example(), names)
    assert names["x"].shape == (4, 7, 24) and names["loss"].shape == ()
    assert float(table.grad.norm()) <= 1.0 + 1e-5
    assert float(names["masters"][0].norm()) <= 1.0 + 1e-5
