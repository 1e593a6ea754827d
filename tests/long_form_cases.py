"""f5hip_set_long_form (attention through the rotary and sliding-window operators inside the sampler) against the CPU oracle with its attention and
its rotary angles restated for windows; run on the host shim (tests/test_long_form.py) and on the GPU (tests/test_gpu_long_form.py).  Tolerances are the ones
tests/test_gpu_parity.py holds the same precision modes to: the operators' own errors (tests/operators_oracle.py) are those of fp32, or of one fp16
rounding of q, k, v and the weights in the fp16 mode."""
import math
import os
import sys
from contextlib import contextmanager

import pytest
import torch
import torch.nn.functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.join(ROOT, "tests"))
from f5_tts_amd import config, synth  # noqa: E402
from oracle import f5_oracle as O  # noqa: E402
from test_gpu_parity import MXTOL, TIGHT, X3TOL, maxerr  # noqa: E402

TOL = {"fp32": TIGHT, "fp16x3": X3TOL, "fp16m": MXTOL, "fp16": 2e-2}


@contextmanager
def windowed_oracle(window, sinks, freqs=None, amplitude=1.0):
    """The oracle with scaled_dot_product_attention seen through the window and, where given, other rotary angles (64-bit frequencies)."""
    left, right = window
    sdpa, rope, table = F.scaled_dot_product_attention, O.apply_rope, O.rotary_freqs

    def attend(q, k, v, attn_mask=None, dropout_p=0.0, is_causal=False):
        n = q.shape[-2]
        i, j = torch.arange(n)[:, None], torch.arange(n)[None]
        seen = torch.ones(n, n, dtype=torch.bool)
        if right >= 0:
            seen &= j <= i + right
        if left >= 0:
            seen &= (j >= i - left) | (j < sinks)
        if attn_mask is not None:
            seen = seen & attn_mask
        s = (q @ k.transpose(-1, -2) / math.sqrt(q.shape[-1])).masked_fill(~seen, -math.inf)
        return torch.softmax(s, -1).masked_fill(~seen.any(-1, keepdim=True), 0.0) @ v

    def angles(dim_head, n):
        f = torch.arange(n).double()[:, None] * freqs
        return torch.stack((f, f), -1).reshape(1, n, dim_head)

    O.F.scaled_dot_product_attention = attend
    if freqs is not None:
        O.rotary_freqs = angles
        O.apply_rope = lambda t, f: (rope(t.double(), f) * amplitude).to(t.dtype)
    try:
        yield
    finally:
        O.F.scaled_dot_product_attention, O.apply_rope, O.rotary_freqs = sdpa, rope, table


def inputs(preset, batch=1, frames=(90,)):
    cfg = config.PRESETS[preset]
    wav = synth.synth_wave(256 * 20, seed=3, batch=batch)
    text = synth.synth_text_ids(batch, 20, cfg.text_num_embeds, seed=2)
    dur = frames[0] if batch == 1 else torch.tensor(frames)
    return cfg, wav, text, dur, dict(steps=4, cfg_strength=2.0, sway_sampling_coef=-1.0, seed=7)


def check_windows(engines, preset, prec, window, sinks, *, batch=1, frames=(90,), rope=None):
    from f5_tts_amd.engine import F5HipCFM

    eng = engines(preset, 1)
    cfg, wav, text, dur, kw = inputs(preset, batch, frames)
    sd = synth.synth_dit_state_dict(cfg, seed=1)
    freqs, amplitude = None, 1.0
    if rope:
        from f5_tts_amd import ops

        freqs, amplitude = ops.rotary_frequencies(64, scaling=rope[0], factor=rope[1], original_length=rope[2])
    with windowed_oracle(window, sinks, freqs, amplitude):
        ref, _ = O.cfm_sample(sd, cfg, wav, text, dur, **kw)
    eng.set_long_form(window, sinks, **(dict(rope_scaling=rope[0], rope_factor=rope[1], rope_original_length=rope[2]) if rope else {}))
    try:
        out, _ = F5HipCFM(eng, precision=prec).sample(wav.cuda(), text, dur, **kw)
    finally:
        eng.set_long_form()
    valid = [dur] if batch == 1 else [int(x) for x in dur]
    for b, n in enumerate(valid):
        assert maxerr(out[b, :n], ref[b, :n]) < TOL[prec], (b, maxerr(out[b, :n], ref[b, :n]))
    return out


def check_windows_that_hold_everything(engines, prec):
    """Windows over the whole utterance, no scaling: the ordinary oracle's result; and off again, the ordinary path's bytes."""
    from f5_tts_amd.engine import F5HipCFM

    eng = engines("tiny", 1)
    cfg, wav, text, dur, kw = inputs("tiny")
    ref, _ = O.cfm_sample(synth.synth_dit_state_dict(cfg, seed=1), cfg, wav, text, dur, **kw)
    model = F5HipCFM(eng, precision=prec)
    before, _ = model.sample(wav.cuda(), text, dur, **kw)
    try:
        for window in ((-1, -1), (200, 200)):
            eng.set_long_form(window)
            out, _ = model.sample(wav.cuda(), text, dur, **kw)
            assert maxerr(out, ref) < TOL[prec]
    finally:
        eng.set_long_form()
    after, _ = model.sample(wav.cuda(), text, dur, **kw)
    assert torch.equal(before, after)


def check_graph_and_chains(engines):
    """A captured loop, replayed with other work between, and two concurrent chains give the eager result; changing the window drops the graph."""
    from f5_tts_amd.engine import F5HipCFM

    eng = engines("tiny", 1)
    cfg, wav, text, dur, kw = inputs("tiny", 2, (90, 70))
    model = F5HipCFM(eng, precision="fp16x3")
    try:
        eng.set_long_form(15, 20)
        want, _ = model.sample(wav.cuda(), text, dur, **kw)
        eng.set_option("use_graph", 1)
        for _ in range(3):
            got, _ = model.sample(wav.cuda(), text, dur, **kw)
            assert torch.equal(got, want)
        eng.set_option("branch_streams", 1)
        got, _ = model.sample(wav.cuda(), text, dur, **kw)
        assert maxerr(got, want.cpu()) < TIGHT  # the block GEMMs of half the rows may take other tiles
        eng.set_option("branch_streams", -1)
        eng.set_long_form(7, 20)
        other, _ = model.sample(wav.cuda(), text, dur, **kw)
        assert not torch.equal(other, want)
        eng.set_option("use_graph", 0)
        eager, _ = model.sample(wav.cuda(), text, dur, **kw)
        assert torch.equal(other, eager)
    finally:
        eng.set_option("use_graph", 0)
        eng.set_option("branch_streams", -1)
        eng.set_long_form()


def check_refusals(engines):
    eng = engines("tiny", 1)
    for kw in (dict(sinks=5), dict(window=(-2, 0)), dict(window=4, sinks=-1), dict(window=1 << 30), dict(window=4, rope_scaling="cubic"),
               dict(window=4, rope_scaling="linear", rope_factor=0.0), dict(window=4, rope_scaling="yarn", rope_factor=2.0)):
        with pytest.raises(ValueError):
            eng.set_long_form(**kw)
    with pytest.raises(ValueError):
        engines("tiny_unett", 1).set_long_form(4)
    with pytest.raises(ValueError):
        engines("tiny_qknorm", 1).set_long_form(4)


CASES = {
    "fp32": ("tiny", "fp32", (9, 5), 12, {}),
    "fp16x3": ("tiny", "fp16x3", (9, 5), 12, {}),
    "fp16m": ("tiny", "fp16m", (30, 30), 20, {}),
    "fp16": ("tiny", "fp16", (9, 5), 12, {}),
    "masked_ragged": ("tiny_mask", "fp32", (16, 16), 20, dict(batch=3, frames=(90, 41, 63))),
    "unmasked_ragged": ("tiny", "fp16x3", (16, 16), 20, dict(batch=2, frames=(80, 50))),
    "first_head_rotates": ("tiny_v0", "fp32", (20, 20), 20, {}),
    "linear": ("tiny", "fp32", (40, 40), 20, dict(rope=("linear", 2.0, 0))),
    "yarn": ("tiny", "fp16x3", (40, 40), 20, dict(rope=("yarn", 4.0, 60))),
    "inner_is_not_dim": ("tiny_inner512", "fp16x3", (16, 8), 20, {}),
}
