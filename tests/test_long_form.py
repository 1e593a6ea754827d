"""The sampler's long form on the host shim (tests/long_form_cases.py): the engine's own sources compiled for the CPU."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests"))
import long_form_cases as L  # noqa: E402
from test_hipemu import CLANG, engine_emu_lib  # noqa: E402,F401
from test_parity_on_shim import shim_engines  # noqa: E402,F401

pytestmark = pytest.mark.skipif(not os.path.exists(CLANG), reason="needs the ROCm host clang++")


@pytest.mark.parametrize("name", ["fp32", "fp16x3", "fp16", "masked_ragged", "first_head_rotates", "yarn"])
def test_windows_on_the_shim(shim_engines, name):  # noqa: F811
    preset, prec, window, sinks, kw = L.CASES[name]
    L.check_windows(shim_engines, preset, prec, window, sinks, **kw)


def test_windows_that_hold_everything_on_the_shim(shim_engines):  # noqa: F811
    L.check_windows_that_hold_everything(shim_engines, "fp32")


def test_refusals_on_the_shim(shim_engines):  # noqa: F811
    L.check_refusals(shim_engines)
