"""The post-training example: every stage moves the way it is meant to."""

import importlib.util
import math
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "post_training.py"
    spec = importlib.util.spec_from_file_location("post_training", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_post_training(gpu):
    example = _example()
    losses, rewards, margins = example.main()
    assert all(math.isfinite(x) for c in (losses, rewards, margins) for x in c)
    mean = lambda c: sum(c) / len(c)  # noqa: E731
    assert mean(losses[-5:]) < 0.7 * mean(losses[:5])
    assert mean(rewards[-5:]) > 1.5 * mean(rewards[:5])
    assert abs(margins[0]) < 1e-3  # the policy is the reference
    assert mean(margins[-5:]) > 0.5
