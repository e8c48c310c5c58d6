"""The neural shading example: the surface's ops, group norm and AdamW together."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location(
        "neural_shading", os.path.join(ROOT, "examples", "neural_shading.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_the_shader_learns():
    """From the loss of a random shader, about the colours' variance of 0.1, to a twentieth."""
    losses = _example().train(steps=120, size=96, views=2, level=3)
    first, last = sum(losses[:5]) / 5, sum(losses[-5:]) / 5
    print(f"[neural shading] {first:.4f} -> {last:.4f}", flush=True)
    assert torch.tensor(losses).isfinite().all()
    assert last < first / 20


def test_the_same_seed_learns_the_same():
    """Every sum runs in a fixed order."""
    a, b = (_example().train(steps=5, size=64, views=2, level=2) for _ in range(2))
    assert a == b
