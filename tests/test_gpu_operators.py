"""GPU tests of the operators with entry points of their own (f5-tts_amd/ops.py) against the 64-bit restatement in tests/operators_oracle.py."""
import os
import sys
import threading

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.join(ROOT, "tests"))
import operators_oracle as O  # noqa: E402
from f5_tts_amd import ops  # noqa: E402
from test_operators import check_unseen  # noqa: E402

pytestmark = pytest.mark.gpu


def gpu(t):
    return t.cuda()


@pytest.mark.parametrize("name", sorted(O.ROTARY))
def test_rotary(name):
    O.check_rotary(ops, gpu, O.ROTARY[name])


@pytest.mark.parametrize("dtype", sorted(O.TYPES))
@pytest.mark.parametrize("half", [False, True])
def test_rotary_long(dtype, half):
    """Enough tokens for several heads to a thread; a scaled plan's frequencies and amplitude."""
    b, n, h, hk, d, r = 3, 1406, 16, 4, 64, 48
    g = torch.Generator().manual_seed(3)
    q, k = torch.randn(b, n, h, d, generator=g).to(O.TYPES[dtype]), torch.randn(b, n, hk, d, generator=g).to(O.TYPES[dtype])
    f, a = ops.rotary_frequencies(r, scaling="yarn", factor=4.0, original_length=1024)
    at = torch.randint(0, 1 << 20, (b, n), generator=g)
    got = ops.rotary(q.cuda(), k.cuda(), f.cuda(), amplitude=a, positions=at.cuda(), layout="half" if half else "interleaved")
    for x, y in zip((q, k), got):
        ref, tol = O.rotary(x, f, at, amplitude=a, half=half)
        assert O.over(y, ref, tol) <= 1


def test_rotary_in_place_inverse_and_gradient():
    g = torch.Generator().manual_seed(1)
    fused = torch.randn(2, 300, 24, 64, generator=g).cuda()
    q, k, f = fused[:, :, :16], fused[:, :, 16:20], O.frequencies(64).cuda()
    before = fused.clone()
    apart = ops.rotary(q, k, f, layout="half")
    ops.rotary(q, k, f, layout="half", out=(q, k))
    assert torch.equal(q, apart[0]) and torch.equal(k, apart[1]) and torch.equal(fused[:, :, 20:], before[:, :, 20:])
    ops.rotary(q, k, f, layout="half", inverse=True, out=(q, k))
    # there and back: each way off by at most (2^-22.3 + 2^-22 + 5 2^-24) (|x| + |y|) <= 2^-20 (|x| + |y|)
    size = before[:, :, :16].abs() + before[:, :, :16].roll(32, -1).abs()
    assert ((q - before[:, :, :16]).abs() <= 2 * 2.0 ** -20 * 1.5 * size).all()
    # the gradient of sum(w * rotary(x)) is the inverse call on w, amplitude and all; against central differences in 64 bits
    x, w = torch.randn(1, 3, 1, 8, generator=g), torch.randn(1, 3, 1, 8, generator=g)
    f8 = O.frequencies(8)
    grad = ops.rotary(w.cuda(), None, f8.cuda(), amplitude=1.3, inverse=True, offset=9)[0].cpu().double()
    at = torch.arange(3) + 9
    for i in range(x.numel()):
        e = torch.zeros(x.numel(), dtype=torch.float64)
        e[i] = 0.5
        e = e.view_as(x)
        up, down = ((O.rotary(x.double() + s * e, f8, at, amplitude=1.3)[0] * w.double()).sum() for s in (1, -1))
        # linear, so the difference is exact; the kernel's own error, as above with amplitude 1.3
        assert abs(float(up - down) - float(grad.flatten()[i])) <= 1.3 * 2.0 ** -20 * 2 * float(w.abs().max())


@pytest.mark.parametrize("name", sorted(O.ATTENTION))
def test_window_attention(name):
    O.check_attention(ops, gpu, O.ATTENTION[name])


@pytest.mark.parametrize("case", [
    (2, 1406, 1406, 4, 4, 64, "fp16", 256, 256, 469, "start", None, None),
    (1, 777, 777, 6, 2, 128, "bf16", 300, 0, 17, "start", None, None),
    (1, 500, 500, 2, 2, 64, "fp32", 100, 100, 60, "start", None, None),
    (3, 65, 1500, 8, 2, 128, "bf16", 700, 0, 33, "end", [1500, 900, 10], None),
    (5, 1, 4000, 16, 4, 128, "fp16", 2047, 0, 4, "end", [4000, 1, 0, 2500, 333], None),
    (2, 4, 9000, 8, 1, 64, "bf16", -1, 0, 0, "end", [9000, 5000], [4, 1]),
    (1, 2, 2500, 4, 4, 128, "fp32", 2000, 0, 100, "end", None, None),
    (16, 330, 330, 32, 32, 64, "fp16", 60, 40, 75, "start", [330 - 20 * i for i in range(16)], None),
    (9, 300, 700, 64, 64, 64, "bf16", 90, 0, 5, "end", None, [300 - 35 * i for i in range(9)]),
    (2, 1, 300, 40, 1, 96, "fp16", 250, 0, 9, "end", None, None),
], ids=lambda c: "-".join(map(str, c[:7])))
def test_window_attention_larger(case):
    O.check_attention(ops, gpu, case, seed=5)


@pytest.mark.parametrize("case", [
    (1, 1, 3000, 16, 16, 64, "fp16", -1, 0, 0, "end", None, None),
    (2, 40, 2000, 16, 4, 128, "bf16", 1500, 0, 9, "end", [2000, 1203], [40, 33]),
    (8, 200, 600, 8, 1, 64, "fp16", -1, 0, 0, "end", [600, 200, 0, 599, 1, 64, 65, 333], None),
    (4, 170, 900, 4, 2, 64, "fp32", 700, 30, 20, "start", [900, 170, 20, 450], None),
], ids=lambda c: "-".join(map(str, c[:7])))
def test_window_attention_units_in_turns(case):
    """Whole (sequence, key head) units to each XCD, their blocks in turns, with and without ranges of keys."""
    O.check_attention(ops, gpu, case, seed=6)


@pytest.mark.parametrize("name", ["both_sides", "token_grouped", "fp32_both_sides"])
def test_window_attention_sharp_scores(name):
    """Scores up to a few hundred: one key carries a row, and the running maximum moves by more than the type's range."""
    O.check_attention(ops, gpu, O.ATTENTION[name], seed=2, spread=40.0)
    O.check_attention(ops, gpu, O.ATTENTION[name], seed=3, scale=-1.0)


def test_window_attention_of_huge_scores():
    O.check_huge_scores(ops, gpu)


def test_window_attention_of_a_nan():
    O.check_seen_nan(ops, gpu)


def test_window_attention_ignores_what_nobody_sees():
    check_unseen(ops, gpu)


def test_window_attention_views_and_rows_left_alone():
    g = torch.Generator().manual_seed(7)
    fused = torch.randn(2, 200, 12, 64, generator=g).half().cuda()
    q, k, v = fused[:, :, :6], fused[:, :, 6:9], fused[:, :, 9:]
    kw = dict(window=(31, 12), sinks=5)
    want = ops.window_attention(q.contiguous(), k.contiguous(), v.contiguous(), **kw)
    assert torch.equal(ops.window_attention(q, k, v, **kw), want)
    swapped = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]  # [batch, heads, tokens, head_dim] in memory
    assert torch.equal(ops.window_attention(*swapped, **kw), want)
    odd = torch.randn(2 * 200 * 6 * 64 + 3, generator=g).half().cuda()
    odd = odd[3:].view(2, 200, 6, 64)
    odd.copy_(q)  # not aligned to 16 bytes: copied by the call
    assert torch.equal(ops.window_attention(odd, k, v, **kw), want)
    one = ops.window_attention(q[:1].expand(2, 200, 6, 64), k[:1].expand(2, 200, 3, 64), v[:1].expand(2, 200, 3, 64), **kw)
    assert torch.equal(one[0], want[0]) and torch.equal(one[1], want[0])
    out = torch.full((2, 200, 8, 64), 7.0, dtype=torch.float16, device="cuda")
    lens = torch.tensor([200, 13], dtype=torch.int64, device="cuda")
    ops.window_attention(q, k, v, q_len=lens, out=out[:, :, 1:7], **kw)
    assert torch.equal(out[0, :, 1:7], want[0]) and torch.equal(out[1, :13, 1:7], want[1, :13])
    assert (out[1, 13:] == 7).all() and (out[:, :, 0] == 7).all() and (out[:, :, 7] == 7).all()
    bad = torch.tensor([-5, 100000], dtype=torch.int32, device="cuda")  # clamped into [0, tokens]
    got = ops.window_attention(q, k, v, kv_len=bad, q_len=bad, **kw)
    assert (got[0] == 0).all() and torch.equal(got[1], want[1])


def test_window_attention_far_in_a_long_cache():
    """Keys whose byte offsets pass 32 bits: 40 000 tokens of a cache with 2^17 bytes between them."""
    n, step = 40000, 1 << 16
    cache = torch.empty(n * step, dtype=torch.float16, device="cuda").view(1, n, step)
    k, v = cache[:, :, :128].view(1, n, 2, 64), cache[:, :, 128:256].view(1, n, 2, 64)
    g = torch.Generator().manual_seed(9)
    hk, hv, q = (torch.randn(1, m, 2, 64, generator=g).half() for m in (300, 300, 70))
    k[:, -300:], v[:, -300:] = hk.cuda(), hv.cuda()
    ref, tol, _ = O.attention(q, hk, hv, window=(200, 0), align="end")
    for m in (70, 1):  # the form for many rows and the one for few
        out = ops.window_attention(q[:, -m:].cuda(), k, v, window=(200, 0), align="end")
        assert O.over(out, ref[:, -m:], tol[:, -m:]) <= 1


def test_streams_threads_and_graphs():
    g = torch.Generator().manual_seed(11)
    f = O.frequencies(64).cuda()
    sets = [[torch.randn(2, m, h, 64, generator=g).half().cuda() for m, h in ((3, 8), (900, 2), (900, 2))] for _ in range(4)]

    def step(q, k, v):
        q, _ = ops.rotary(q, None, f, offset=897)
        return ops.window_attention(q, ops.rotary(k, None, f)[0], v, window=(600, 0), sinks=4, align="end")

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    got, streams = [None] * 4, [torch.cuda.Stream() for _ in range(4)]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(5):
                got[i] = step(*sets[i])

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # two graphs, replayed side by side and with eager calls between the replays
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*sets[i]))
        graphs.append(graph)
    for _ in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        eager = step(*sets[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])
    sets[0][0].mul_(0.5)  # a replay reads its inputs anew
    fresh = step(*sets[0])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], fresh) and not torch.equal(fresh, want[0])
