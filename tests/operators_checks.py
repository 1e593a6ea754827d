"""More cases of the operators that the CPU (host shim) and GPU tests share; tests/operators_oracle.py has the definitions in 64 bits."""
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
