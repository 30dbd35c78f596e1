"""The example that trains a token policy and verifies it, end to end: what the policy answers rightly
rises from chance, and part of it is certified."""

import importlib.util
import math
import os

import pytest

from tests.gpu_util import announce, device

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_train_and_verify():
    device()
    spec = importlib.util.spec_from_file_location("train_and_verify", os.path.join(ROOT, "examples", "train_and_verify.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.main(["--steps", "60", "--contexts", "256", "--eps", "0.02"])
    (right0, certified0, _), (right1, certified1, margin1) = got["before"], got["after"]
    announce(f"right {right0:.3f} -> {right1:.3f}, certified {certified0:.3f} -> {certified1:.3f}, losses {got['losses']}")
    assert all(math.isfinite(x) for x in got["losses"])
    # 256 contexts, 8 actions: chance is an eighth; the table and the MLP have 20 parameters a context
    assert right0 < 0.4 and right1 > 0.9
    assert certified1 > 0.5 and certified1 > certified0 and certified1 <= right1
