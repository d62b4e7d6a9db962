"""The operators together, as a training program uses them: the example's student under the engine."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("distill_student", os.path.join(ROOT, "examples", "distill_student.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_student_learns(example):
    losses = example.train(25)
    assert losses.isfinite().all()
    assert losses[-1] < 0.6 * losses[0], losses


def test_the_scale_told_ahead_changes_nothing(example):
    """The same gradients, made in the forward pass or in the backward pass: the logits' are the same numbers rounded once, and what torch
    makes of them is too, except where its own kernels add in another order from run to run (2**-10 of the loss after three steps)."""
    a, b = example.train(4, ahead=True), example.train(4, ahead=False)
    assert torch.equal(a[0], b[0])
    assert ((a - b).abs() <= 2.0**-10 * a.abs()).all(), (a, b)
