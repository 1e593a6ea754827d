"""The sampler's long form as two concurrent chains, long enough that each keeps partial results of its own in the workspace."""
import ctypes as C
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.join(ROOT, "tests"))
import long_form_cases as L  # noqa: E402
from f5_tts_amd import binding, config, ops  # noqa: E402
from test_gpu_parity import TIGHT, engines, maxerr  # noqa: E402,F401  (the fixture)

pytestmark = pytest.mark.gpu
WINDOW, SINKS, FRAMES = (500, 450), 40, (1500, 1201)


def workspace(batch, n, heads, dtype):
    """Bytes that one attention launch of a chain needs; the pointers are nobody's memory, nothing is launched."""
    st = [3 * heads * 64 * n, 3 * heads * 64, 64] * 3 + [heads * 64 * n, heads * 64, 64]
    at = [1 << (40 + i) for i in range(4)]
    args = ops._WINDOW.pack(dtype, batch, n, n, heads, heads, 64, *WINDOW, SINKS, 0, 0.125, *at, *st, 0, 0, 0, 0)
    return binding.load_library().f5hip_window_attention_workspace(args)


@pytest.mark.parametrize("prec", ["fp32", "fp16x3", "fp16"])
@pytest.mark.parametrize("frames", [FRAMES[:1], FRAMES])
def test_chains_with_partial_results(engines, prec, frames):  # noqa: F811
    from f5_tts_amd.engine import F5HipCFM

    eng, batch = engines("tiny", 1), len(frames)
    heads = config.PRESETS["tiny"].heads
    assert workspace(batch, max(frames), heads, 1 if prec == "fp16" else 0) > 0
    _, wav, text, dur, kw = L.inputs("tiny", batch, frames)
    model = F5HipCFM(eng, precision=prec)
    outs = []
    try:
        eng.set_long_form(WINDOW, SINKS)
        for chains, graph in ((0, 0), (1, 0), (1, 1), (1, 1)):
            eng.set_option("branch_streams", chains)
            eng.set_option("use_graph", graph)
            outs.append(model.sample(wav.cuda(), text, dur, **kw)[0].cpu())
    finally:
        eng.set_option("branch_streams", -1)
        eng.set_option("use_graph", 0)
        eng.set_long_form()
    for out in outs[1:]:
        for b, n in enumerate(frames):
            # the block GEMMs of half the rows may take other tiles, and the key ranges of half the sequences be others
            assert maxerr(out[b, :n], outs[0][b, :n]) < (TIGHT if prec != "fp16" else L.TOL["fp16"])
    assert torch.equal(outs[1], outs[2]) and torch.equal(outs[1], outs[3])
