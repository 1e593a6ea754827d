"""The sampler's long form on the GPU (tests/long_form_cases.py)."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests"))
import long_form_cases as L  # noqa: E402
from test_gpu_parity import engines  # noqa: E402,F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", sorted(L.CASES))
def test_windows(engines, name):  # noqa: F811
    preset, prec, window, sinks, kw = L.CASES[name]
    L.check_windows(engines, preset, prec, window, sinks, **kw)


@pytest.mark.parametrize("prec", ["fp32", "fp16x3", "fp16m", "fp16"])
def test_windows_that_hold_everything(engines, prec):  # noqa: F811
    L.check_windows_that_hold_everything(engines, prec)


def test_graph_and_chains(engines):  # noqa: F811
    L.check_graph_and_chains(engines)


def test_refusals(engines):  # noqa: F811
    L.check_refusals(engines)


def test_a_long_utterance(engines):  # noqa: F811
    """1500 frames: many row blocks and key tiles a launch, the prompt as sinks."""
    L.check_windows(engines, "tiny", "fp32", (100, 100), 40, frames=(1500,))
    L.check_windows(engines, "tiny", "fp16x3", (100, 100), 40, frames=(1500,), rope=("ntk", 2.0, 0))
