"""The example's training step: the operators together, in place and strided."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_the_student_learns():
    path = Path(__file__).resolve().parent.parent / "examples" / "attention_entry_step.py"
    spec = importlib.util.spec_from_file_location("attention_entry_step", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses = mod.train(30, report=lambda line: None)
    assert all(torch.isfinite(torch.tensor(losses)))
    assert losses[-1] < 0.5 * losses[0]
