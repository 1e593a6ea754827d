"""GPU tests of the operators at the ends of their ranges (tests/operators_checks.py)."""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.join(ROOT, "tests"))
import operators_checks as K  # noqa: E402
import operators_oracle as O  # noqa: E402
from f5_tts_amd import ops  # noqa: E402

pytestmark = pytest.mark.gpu


def gpu(t):
    return t.cuda()


@pytest.mark.parametrize("name", sorted(K.MORE_ATTENTION))
def test_more_window_attention(name):
    O.check_attention(ops, gpu, K.MORE_ATTENTION[name], seed=8)
    O.check_attention(ops, gpu, K.MORE_ATTENTION[name], seed=9, spread=30.0)


def test_window_attention_of_large_values():
    K.check_large_values(ops, gpu)


def test_window_attention_of_nan_keys():
    K.check_nan_keys(ops, gpu)


def test_rotary_of_far_positions():
    K.check_far_positions(ops, gpu)
