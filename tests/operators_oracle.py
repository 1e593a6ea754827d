"""64-bit restatements of the operators (include/f5hip.h, "operators"), their error bounds, and the cases that the CPU (host shim) and GPU
tests share.  A rounding to type t is off by at most u = finfo(t).eps / 2, relative to the value."""
import math

import torch

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def half_step(t):
    return torch.finfo(t).eps / 2


def frequencies(rot, base=10000.0):
    return base ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)


def rotary(x, freq, positions, *, amplitude=1.0, half=False, heads=None, inverse=False):
    """([B, T, H, D] in 64 bits, its error bound): x any dtype, positions int64 [B, T] or [T]."""
    r, y = 2 * freq.shape[0], x.double().clone()
    angle = positions.double()[..., None, None] * freq
    if angle.dim() == 3:
        angle = angle[None]
    c, s = torch.cos(angle) * amplitude, torch.sin(angle) * amplitude * (-1 if inverse else 1)
    a, b = (slice(0, r // 2), slice(r // 2, r)) if half else (slice(0, r, 2), slice(1, r, 2))
    n = x.shape[2] if heads is None else min(heads, x.shape[2])
    u, v = x[:, :, :n, a].double(), x[:, :, :n, b].double()
    y[:, :, :n, a], y[:, :, :n, b] = u * c - v * s, u * s + v * c
    # one rounding of the output; cos and sin: 2^-25 turns of the reduced angle = 2^-22.3, two units of the fp32 function = 2^-22, the
    # amplitude, two products and a sum, 2^-24 each; the 64-bit angle, on both sides, p f 2^-52
    fp32 = 2.0 ** -22.3 + 2.0 ** -22 + 4 * 2.0 ** -24 + float(positions.double().abs().max() if positions.numel() else 0) * 2.0 ** -51
    tol = torch.zeros_like(y)
    tol[:, :, :n, :r] = half_step(x.dtype) * y[:, :, :n, :r].abs()
    size = (u.abs() + v.abs()) * abs(amplitude) * fp32
    tol[:, :, :n, a] += size
    tol[:, :, :n, b] += size
    if x.dtype == torch.float16:
        tol[:, :, :n, :r] += 2.0 ** -25  # half a step among the subnormal numbers
    return y, tol


def attention(q, k, v, *, window=(-1, -1), sinks=0, kv_len=None, q_len=None, align="start", scale=None):
    """(out [B, Tq, H, D] in 64 bits, its error bound, rows [B, Tq] that the operator writes)."""
    b, tq, h, d = q.shape
    tk, hk = k.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    left, right = window
    out, tol = torch.zeros(b, tq, h, d, dtype=torch.float64), torch.zeros(b, tq, h, d, dtype=torch.float64)
    rows = torch.zeros(b, tq, dtype=torch.bool)
    ut, up = half_step(q.dtype), 0.0 if q.dtype == torch.float32 else half_step(q.dtype)
    for i in range(b):
        n = tk if kv_len is None else min(max(int(kv_len[i]), 0), tk)
        m = tq if q_len is None else min(max(int(q_len[i]), 0), tq)
        rows[i, :m] = True
        if not n or not m:
            continue
        p = torch.arange(m)[:, None] + (0 if align == "start" else n - m)
        j = torch.arange(n)[None]
        seen = torch.ones(m, n, dtype=torch.bool)
        if right >= 0:
            seen &= j <= p + right
        if left >= 0:
            seen &= (j >= p - left) | (j < sinks)
        for head in range(h):
            g = head // (h // hk)
            x, y, z = q[i, :m, head].double(), k[i, :n, g].double(), v[i, :n, g].double()
            # what no query sees, or a query does not see, may hold anything
            y, z = (torch.where(torch.isfinite(t), t, torch.zeros_like(t)) for t in (y, z))
            s = (x @ y.T * scale).masked_fill(~seen, -math.inf)
            w = torch.softmax(s, -1).masked_fill(~seen.any(-1, keepdim=True), 0.0)
            o, mass = w @ z, w @ z.abs()
            out[i, :m, head] = o
            # the scores: d products summed in fp32, one rounding of scale log2(e) and one of the scaled score, the exponential's own 2^-22
            big = ((x.abs() @ y.abs().T) * abs(scale)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            ds = big * (d + 4) * 2.0 ** -24 + 2.0 ** -22
            # each weight is off by e^ds - 1 and, in 16 bits, by its rounding; the sums over n keys by 2^-24 a step (two sums, and a merge
            # of parts); numerator and denominator each, hence mass + |o|; then the output's own rounding
            dw = torch.expm1(ds) + up + (n + 16) * 2.0 ** -24
            tol[i, :m, head] = dw * (mass + o.abs()) * (1 + 2 * up) + ut * o.abs()
            if q.dtype == torch.float16:
                # half a step among the subnormal numbers, 2^-25: of the output, and of each weight, which are held so that the row's
                # largest is at least 2^7 (and their sum with it): 2^-32 of |v| for every key seen, in numerator and denominator
                tol[i, :m, head] += 2.0 ** -25 + 2.0 ** -32 * (seen.double() @ z.abs() + seen.sum(-1, keepdim=True) * o.abs())
    return out, tol, rows


def over(x, ref, tol):
    """How far x is from ref, in units of the bound (at most 1 is right)."""
    x = x.detach().cpu().double()
    assert torch.isfinite(x).all()
    d = (x - ref).abs()
    return float(torch.where(d == 0, torch.zeros_like(d), d / tol.clamp_min(1e-300)).max()) if d.numel() else 0.0


# name: (batch, tokens, heads, kv_heads, dim, rot, dtype, half, rot_heads, first, inverse)
ROTARY = {
    "one_token": (1, 1, 4, 4, 64, 64, "fp16", False, None, 131071, False),
    "no_k": (2, 3, 3, 0, 64, 64, "bf16", False, None, 5, False),
    "interleaved_fp32": (2, 17, 4, 2, 64, 64, "fp32", False, None, 0, False),
    "half_fp32": (1, 9, 2, 2, 32, 32, "fp32", True, None, 7, False),
    "half_part_bf16": (2, 33, 8, 2, 128, 96, "bf16", True, None, 0, False),
    "interleaved_part": (1, 5, 3, 1, 80, 32, "fp16", False, None, 1000000, False),
    "half_narrow": (1, 11, 5, 1, 40, 20, "fp16", True, None, 3, False),
    "half_odd_pairs": (1, 4, 2, 1, 30, 10, "bf16", True, None, 3, False),
    "half_single_columns": (2, 3, 2, 1, 7, 6, "fp16", True, None, 3, False),
    "interleaved_single_columns": (2, 3, 2, 1, 9, 6, "fp32", False, None, 3, False),
    "first_head": (2, 6, 4, 4, 64, 64, "fp32", False, 1, 0, False),
    "no_head": (1, 4, 2, 2, 64, 64, "fp16", True, 0, 0, False),
    "inverse": (1, 8, 2, 2, 64, 48, "fp16", True, None, 100, True),
    "negative_positions": (1, 8, 2, 2, 64, 64, "fp32", False, None, -5, False),
    "far": (1, 3, 2, 2, 64, 64, "fp32", True, None, (1 << 31) - 1, False),
    "many_heads": (1, 2, 20, 5, 64, 64, "bf16", True, None, 12, False),
}

# name: (batch, tq, tk, heads, kv_heads, dim, dtype, left, right, sinks, align, kv_len, q_len)
ATTENTION = {
    "one_key": (1, 1, 1, 2, 2, 64, "fp16", 4, 0, 0, "end", None, None),
    "no_keys": (2, 3, 0, 2, 1, 64, "bf16", 4, 0, 1, "start", None, None),
    "token": (2, 1, 150, 4, 4, 64, "fp16", 100, 0, 4, "end", None, None),
    "token_grouped": (3, 1, 300, 8, 2, 128, "bf16", 70, 0, 3, "end", [300, 0, 77], None),
    "token_all": (1, 1, 333, 4, 1, 64, "fp16", -1, -1, 0, "end", [200], None),
    "token_fp32": (2, 1, 140, 4, 2, 64, "fp32", 64, 0, 5, "end", [140, 66], None),
    "three_tokens_odd_group": (2, 3, 90, 6, 2, 40, "bf16", 30, 0, 2, "end", [90, 2], None),
    "chunk": (2, 20, 200, 4, 2, 64, "fp16", 63, 0, 7, "end", [200, 31], None),
    "chunk_ragged": (3, 9, 100, 4, 2, 96, "bf16", 40, 0, 5, "end", [100, 5, 50], [9, 4, 0]),
    "chunk_longer_than_keys": (1, 12, 7, 2, 2, 64, "fp16", 3, 0, 1, "end", None, None),
    "both_sides": (1, 150, 150, 2, 2, 64, "fp16", 20, 30, 40, "start", None, None),
    "both_sides_bf16_128": (1, 130, 130, 2, 1, 128, "bf16", 33, 17, 3, "start", None, None),
    "both_sides_96": (1, 70, 70, 2, 1, 96, "fp16", 12, 30, 3, "start", None, None),
    "both_sides_40": (1, 70, 90, 3, 1, 40, "bf16", 50, 3, 20, "start", None, None),
    "fp32_96": (1, 50, 90, 3, 1, 96, "fp32", 50, 3, 20, "end", None, None),
    "causal": (1, 97, 97, 2, 2, 64, "bf16", -1, 0, 0, "start", None, None),
    "full": (1, 70, 70, 2, 2, 64, "fp16", -1, -1, 0, "start", None, None),
    "fp32_both_sides": (1, 140, 140, 2, 2, 64, "fp32", 25, 25, 30, "start", None, None),
    "fp32_odd_dim": (1, 33, 40, 2, 1, 36, "fp32", 9, 4, 2, "start", None, None),
    "fp32_128": (1, 66, 66, 2, 1, 128, "fp32", 40, 0, 2, "start", None, None),
    "ragged": (4, 75, 75, 2, 2, 64, "fp16", 16, 16, 9, "start", [75, 1, 0, 40], None),
    "window_of_nothing_but_itself": (1, 70, 70, 2, 2, 64, "fp16", 0, 0, 0, "start", None, None),
    "sinks_past_the_end": (1, 50, 50, 2, 2, 64, "fp16", 5, 5, 1000, "start", None, None),
    "queries_past_the_keys": (1, 90, 30, 2, 2, 64, "bf16", 10, 10, 0, "start", None, None),
    "queries_past_the_keys_fp32": (1, 90, 30, 2, 2, 64, "fp32", 10, 10, 3, "start", None, None),
}


def rotary_inputs(case, seed=0):
    b, n, h, hk, d, rot, dtype, half, heads, first, inverse = case
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(b, n, h, d, generator=g).to(TYPES[dtype])
    k = torch.randn(b, n, hk, d, generator=g).to(TYPES[dtype]) if hk else None
    return q, k, frequencies(rot), dict(layout="half" if half else "interleaved", rot_heads=heads, offset=first, inverse=inverse)


def check_rotary(ops, to, case, amplitude=1.0, seed=0):
    q, k, freq, kw = rotary_inputs(case, seed)
    got = ops.rotary(to(q), None if k is None else to(k), to(freq), amplitude=amplitude, **kw)
    at = torch.arange(q.shape[1]) + kw["offset"]
    for x, y in zip((q, k), got):
        if x is None:
            assert y is None
            continue
        ref, tol = rotary(x, freq, at, amplitude=amplitude, half=kw["layout"] == "half", heads=kw["rot_heads"], inverse=kw["inverse"])
        assert y.dtype == x.dtype and y.shape == x.shape
        assert over(y, ref, tol) <= 1


def attention_inputs(case, seed=0, spread=1.0):
    b, tq, tk, h, hk, d, dtype, left, right, sinks, align, kv_len, q_len = case
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(b, tq, h, d, generator=g) * spread).to(TYPES[dtype])
    k, v = (torch.randn(b, tk, hk, d, generator=g).to(TYPES[dtype]) for _ in range(2))
    kw = dict(window=(left, right), sinks=sinks, align=align)
    kw["kv_len"], kw["q_len"] = (None if x is None else torch.tensor(x, dtype=torch.int32) for x in (kv_len, q_len))
    return q, k, v, kw


def check_attention(ops, to, case, seed=0, spread=1.0, scale=None):
    q, k, v, kw = attention_inputs(case, seed, spread)
    ref, tol, rows = attention(q, k, v, scale=scale, **kw)
    on = {x: to(y) if isinstance(y, torch.Tensor) else y for x, y in kw.items()}
    out = ops.window_attention(to(q), to(k), to(v), scale=scale, **on)
    assert out.dtype == q.dtype and out.shape == q.shape
    assert over(out, ref, tol) <= 1
    assert (out.cpu()[~rows] == 0).all()
    return out


def check_huge_scores(ops, to):
    """Scores down to -2 million, each row one-hot by a margin of 32 768: the first key of a row's window.  16-bit types: the weight cancels against
    the sum up to 2^-22 of a 16-bit number, so exactly; fp32: six of nine piece products (2^-21), the division and two products (2^-23 each)."""
    for dtype in ("bf16", "fp16", "fp32"):
        for n, m in ((70, 70), (70, 2)):
            q = torch.full((1, m, 2, 64), 2.0 ** 6).to(TYPES[dtype])
            k = (-(torch.arange(n) + 1.0) * 2.0 ** 6)[None, :, None, None].expand(1, n, 2, 64).contiguous().to(TYPES[dtype])
            v = torch.randn(1, n, 2, 64, generator=torch.Generator().manual_seed(1)).to(TYPES[dtype])
            out = ops.window_attention(to(q), to(k), to(v), window=(20, 0), align="end").cpu()
            first = (torch.arange(m) + n - m - 20).clamp_min(0)
            if dtype == "fp32":
                assert torch.allclose(out[0], v[0, first], rtol=2.0 ** -20, atol=0)
            else:
                assert torch.equal(out[0], v[0, first])


def check_seen_nan(ops, to):
    """A NaN that a row sees is its result, whatever form the sizes take; a row of q reaches no other row."""
    for name in ("token_fp32", "token_grouped", "three_tokens_odd_group", "chunk", "both_sides", "fp32_both_sides", "both_sides_bf16_128"):
        q, k, v, kw = attention_inputs(ATTENTION[name])
        ref, tol, rows = attention(q, k, v, **kw)
        q[0, -1, 1] = math.nan
        out = ops.window_attention(to(q), to(k), to(v), **{x: to(y) if isinstance(y, torch.Tensor) else y for x, y in kw.items()}).cpu()
        assert out[0, -1, 1].isnan().all()
        out[0, -1, 1] = ref[0, -1, 1].to(out.dtype)
        assert over(out, ref, tol) <= 1
