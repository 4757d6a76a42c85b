"""The integration guide's example of the operators on dense rows: its calls fit the functions'
parameters, and it runs as printed."""

import ast
import inspect
import re
from pathlib import Path

import pytest
import torch

import nacho_amd

GUIDE = Path(__file__).resolve().parent.parent / "INTEGRATION.md"


def _example():
    section = GUIDE.read_text().split("## 3b.")[1].split("\n## ")[0]
    return re.search(r"```python\n(.*?)```", section, re.S).group(1)


def test_calls_fit_the_parameters():
    calls = [n for n in ast.walk(ast.parse(_example())) if isinstance(n, ast.Call)]
    assert len(calls) == 7
    for call in calls:
        named = {x.arg: None for x in call.keywords}
        inspect.signature(getattr(nacho_amd, call.func.attr)).bind(*call.args, **named)


@pytest.mark.gpu
def test_example_runs(gpu):
    def normal(*shape):
        return torch.randn(*shape, device=gpu).requires_grad_()

    keys, n_experts = 1500, 4
    names = {"nacho": nacho_amd, "keys": keys, "n_experts": n_experts,
             "q": normal(2, 9, 8, 64), "k": normal(2, keys, 2, 64), "v": normal(2, keys, 2, 64),
             "lengths": torch.tensor([keys, 700], dtype=torch.int32, device=gpu),
             "experts": torch.randint(0, n_experts, (18, 2), device=gpu),
             "x": normal(18, 32), "expert_rows": normal(36, 32), "weights": normal(18, 2)}
    exec(_example(), names)
    assert names["blocks"].shape == (2, 9, 2, 16) and names["blocks"].dtype == torch.int32
    assert names["out"].shape == (2, 9, 8, 64) and names["y"].shape == (18, 32)
    total = names["out"].sum() + names["rows"].sum() + names["y"].sum()
    total.backward()
    for x in ("q", "k", "v", "x", "expert_rows", "weights"):
        assert torch.isfinite(names[x].grad).all(), x
