"""The example network trains through the attention kernels and its scores are solved."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "match_points.py"


def test_example_learns_to_match(device):
    spec = importlib.util.spec_from_file_location("match_points", EXAMPLE)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, right = example.train(steps=60, pairs=4, points=48, log=lambda _: None)
    # chance: a loss of 2 log 48 = 7.7 and one point in 48
    assert losses[0] > 5.0 and sum(losses[-5:]) / 5 < losses[0] / 2
    assert right > 0.5
