"""More cases of the operators that the CPU (host shim) and GPU tests share; tests/operators_oracle.py has the definitions in 64 bits."""
import math
from fractions import Fraction

import operators_oracle as O
import torch


def check_large_values(ops, to):
    """Values near the largest that the sums hold (16 |v| keys below 2^128): the first 64 keys at score 0, the others higher by less and by more than
    what raises the softmax's reference.  Every value of a column is the same, so the result is that value: sums over n keys in numerator and
    denominator are off by (n + 16) 2^-24 each, the division and the products by 2^-22, bf16 by its own rounding."""
    for dtype in ("fp32", "bf16"):
        t = O.TYPES[dtype]
        for rows, n, heads, d in ((1, 240, 1, 64), (1, 2100, 1, 64), (40, 240, 1, 64), (40, 240, 1, 128), (3, 240, 4, 96), (70, 2100, 1, 128)):
            for above in (6.5, 2.6875, 1.0, 20.0):
                value = torch.tensor([2.0 ** 128 / (17 * n), -1e34, 1e30, 1.0]).to(t)
                q, k = torch.zeros(1, rows, heads, d, dtype=t), torch.zeros(1, n, 1, d, dtype=t)
                q[..., 0] = 1
                k[:, 64:, :, 0] = above
                v = value.repeat(d // 4).expand(1, n, 1, d).contiguous()
                out = ops.window_attention(to(q), to(k), to(v), scale=1.0).cpu().double()
                assert torch.isfinite(out).all(), (dtype, rows, n, above)
                want = v[0, 0, 0].double()
                rel = 2 * (n + 16) * 2.0 ** -24 + 2.0 ** -22 + (O.half_step(t) if dtype == "bf16" else 0)
                assert ((out - want).abs() <= rel * want.abs()).all(), (dtype, rows, n, above)


def exact_turn(p, f):
    """(cos, sin) of the angle p f, p a whole number and f a 64-bit float, both exact: reduced as a fraction of a turn with 1 / 2 pi to 400 bits."""
    r = Fraction(p) * Fraction(f) * TURN
    r = float(r - round(r))
    return math.cos(2 * math.pi * r), math.sin(2 * math.pi * r)


def _turn(bits=400):
    def arctan_of_inverse(x):
        total = term = (1 << bits) // x
        n = 1
        while term:
            n, term = n + 2, -term // (x * x)
            total += term // n
        return total

    # pi / 4 = 4 arctan(1 / 5) - arctan(1 / 239)
    return Fraction(1 << bits, 8 * (4 * arctan_of_inverse(5) - arctan_of_inverse(239)))


TURN = _turn()


def check_far_positions(ops, to):
    """Angles are those of the exact product up to 2^53: the fp32 terms of operators_oracle.rotary's bound, without one that grows with the position."""
    far = [0, 1, -3, 131071, 2 ** 31 - 1, -2 ** 31, 2 ** 37 + 12345, 2 ** 40, -2 ** 45 + 7, 2 ** 50 + 1, 2 ** 53, -2 ** 53]
    for rot, base in ((64, 10000.0), (8, 500000.0)):
        f = O.frequencies(rot, base)
        at = torch.tensor(far)
        turns = [[exact_turn(p, float(x)) for x in f] for p in far]
        c, s = (torch.tensor([[t[i] for t in row] for row in turns], dtype=torch.float64) for i in (0, 1))
        x = torch.randn(1, len(far), 1, rot, generator=torch.Generator().manual_seed(3))
        u, v = x.double()[0, :, 0, 0::2], x.double()[0, :, 0, 1::2]
        size = (u.abs() + v.abs()) * (2.0 ** -22.3 + 2.0 ** -22 + 4 * 2.0 ** -24)
        runs = [ops.rotary(to(x), None, to(f), positions=to(at))[0]]
        runs.append(torch.cat([ops.rotary(to(x[:, i:i + 1]), None, to(f), offset=p)[0] for i, p in enumerate(far)], 1))
        for y in runs:
            y = y.cpu().double()[0, :, 0]
            for got, want in ((y[:, 0::2], u * c - v * s), (y[:, 1::2], u * s + v * c)):
                assert ((got - want).abs() <= size + 2.0 ** -24 * want.abs()).all(), rot


# forms that operators_oracle.ATTENTION does not reach: 32 bits at up to 64 columns in 1024 and more blocks of 128 rows (32-key tiles in two stages),
# few rows at 96 columns in fp32 and fp16, with one range of keys and with several
MORE_ATTENTION = {
    "fp32_many_blocks": (16, 140, 140, 32, 32, 64, "fp32", 30, 5, 9, "start", None, None),
    "fp32_many_blocks_grouped": (9, 70, 90, 128, 64, 36, "fp32", 40, 3, 2, "end", [90 - 11 * i for i in range(9)], [70, 70, 1, 0, 33, 70, 64, 65, 2]),
    "few_rows_fp32_96": (2, 1, 300, 6, 2, 96, "fp32", 250, 0, 9, "end", [300, 41], None),
    "few_rows_fp16_96": (2, 3, 300, 6, 2, 96, "fp16", 250, 0, 9, "end", [300, 41], [3, 2]),
    "few_rows_fp32_96_ranges": (1, 1, 1700, 4, 2, 96, "fp32", -1, 0, 0, "end", None, None),
    "few_rows_fp16_72_ranges": (1, 2, 1700, 4, 2, 72, "fp16", 1600, 0, 3, "end", [1650], None),
}


def check_nan_keys(ops, to):
    """A key that is NaN makes NaN of the rows that see it and touches no other, also those that share its tiles."""
    for name in ("token_grouped", "three_tokens_odd_group", "chunk", "both_sides", "both_sides_bf16_128", "fp32_both_sides", "fp32_odd_dim", "causal"):
        q, k, v, kw = O.attention_inputs(O.ATTENTION[name])
        ref, tol, rows = O.attention(q, k, v, **kw)
        n = k.shape[1] if kw["kv_len"] is None else int(kw["kv_len"][0])
        j = n - 10 if kw["align"] == "end" else (2 * n) // 3  # (a key that some row sees)
        k[0, j] = math.nan
        out = ops.window_attention(to(q), to(k), to(v), **{x: to(y) if isinstance(y, torch.Tensor) else y for x, y in kw.items()}).cpu()
        p = torch.arange(q.shape[1]) + (0 if kw["align"] == "start" else n - q.shape[1])
        left, right = kw["window"]
        sees = torch.ones(q.shape[1], dtype=torch.bool) if right < 0 else j <= p + right
        if left >= 0:
            sees = sees & ((j >= p - left) | (j < kw["sinks"]))
        assert out[0, sees].isnan().all() and sees.any() and (name in ("token_grouped", "three_tokens_odd_group") or not sees.all()), name
        out[0, sees] = ref[0, sees].to(out.dtype)
        assert O.over(out, ref, tol) <= 1, name
