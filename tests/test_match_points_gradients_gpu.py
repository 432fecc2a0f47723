"""The example network's gradients, through every attention entry point, against differences."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "match_points.py"


@pytest.mark.parametrize("training", [False, True])
def test_gradients_of_the_example(device, training):
    """Along a random way, two steps apart: the finer difference is off by a third of what the two
    differ by (h^2 terms), taken whole, and by the loss's float32 roundings over h."""
    spec = importlib.util.spec_from_file_location("match_points", EXAMPLE)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(0)
    model = example.Matcher(16).to(device).train(training)
    *batch, truth = example.sample(2, 40, 16, torch.Generator().manual_seed(0), device)

    def loss():
        scores = model(*batch, seed=5).double()
        log_p = scores.log_softmax(2) + scores.log_softmax(1)
        return -log_p.gather(2, truth[..., None]).mean()

    value = loss()
    grads = torch.autograd.grad(value, list(model.parameters()))
    assert all(g.isfinite().all() and g.any() for g in grads)
    ways = [torch.randn_like(p) * p.detach().std().nan_to_num(0.1).clamp(min=0.01)
            for p in model.parameters()]
    told = sum((g.double() * w.double()).sum() for g, w in zip(grads, ways))

    def slope(h):
        ends = []
        for sign in (1, -1):
            with torch.no_grad():
                for p, w in zip(model.parameters(), ways):
                    p.add_(w, alpha=sign * h)
                ends.append(loss())
                for p, w in zip(model.parameters(), ways):
                    p.sub_(w, alpha=sign * h)
        return (ends[0] - ends[1]) / (2 * h)

    h = 2.0**-7
    wide, fine = slope(2 * h), slope(h)
    # a score is good to a few hundred float32 roundings of its size, 20 at most
    assert (fine - told).abs() <= (wide - fine).abs() + 512 * 2.0**-24 * 20 / h
