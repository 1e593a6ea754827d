"""CPU tests of the operators with entry points of their own (f5-tts_amd/ops.py): frequencies, every refusal, and the kernels' own source on the
host shim (tests/hipemu) against the 64-bit restatement in tests/operators_oracle.py."""
import ctypes as C
import math
import os
import random
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.join(ROOT, "tests"))
import operators_checks as K  # noqa: E402
import operators_oracle as O  # noqa: E402
from f5_tts_amd import binding, ops  # noqa: E402
import hipemu_build  # noqa: E402

CLANG = hipemu_build.CLANG
shim = pytest.mark.skipif(not os.path.exists(CLANG), reason="needs the ROCm host clang++")


@pytest.fixture(scope="module")
def operators_emu_lib():
    lib = C.CDLL(hipemu_build.ensure_operators(), mode=C.RTLD_LOCAL)
    for name, (res, args) in binding.SYMBOLS.items():
        if hasattr(lib, name):
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
    return lib


@pytest.fixture()
def host(operators_emu_lib, monkeypatch):
    """ops over the emulated library: CPU tensors are its device tensors."""
    monkeypatch.setattr(ops, "load_library", lambda *a, **k: operators_emu_lib)
    monkeypatch.setattr(ops, "_device", lambda t: (0, 0))
    return ops


def same(t):
    return t


# ---- frequencies -----------------------------------------------------------------------------------------------------------------------
def test_frequencies_by_their_formulas():
    # pow in 64 bits is within a few units of 2^-53 on either side
    for rot in (2, 64, 96, 128):
        f, a = ops.rotary_frequencies(rot)
        assert a == 1.0 and f.dtype == torch.float64
        assert torch.allclose(f, O.frequencies(rot), rtol=2.0 ** -48, atol=0)
    f0 = O.frequencies(64)
    f, a = ops.rotary_frequencies(64, scaling="linear", factor=4.0)
    assert a == 1.0 and torch.allclose(f, f0 / 4, rtol=2.0 ** -48, atol=0)
    f, a = ops.rotary_frequencies(64, scaling="ntk", factor=2.0)
    assert a == 1.0 and torch.allclose(f, f0 * 2.0 ** (-2.0 * torch.arange(32, dtype=torch.float64) / 62), rtol=2.0 ** -47, atol=0)
    assert f[0] == 1.0  # the fastest frequency stays, the slowest is divided by the factor
    assert math.isclose(f[-1] * 2.0, f0[-1], rel_tol=2.0 ** -47)
    f, a = ops.rotary_frequencies(64, scaling="yarn", factor=8.0, original_length=2048)
    turns = 2048 * f0 / (2 * math.pi)
    assert math.isclose(a, 0.1 * math.log(8.0) + 1)
    assert torch.allclose(f[turns > 32], f0[turns > 32], rtol=2.0 ** -48) and torch.allclose(f[turns < 1], f0[turns < 1] / 8, rtol=2.0 ** -48)
    between = (turns > 1) & (turns < 32)
    assert between.any() and (f[between] < f0[between]).all() and (f[between] > f0[between] / 8).all()


@pytest.mark.parametrize("kw", [dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=-2), dict(rot_dim=64, base=0.0), dict(rot_dim=64, base=float("nan")),
                                dict(rot_dim=64, scaling="cubic"), dict(rot_dim=64, scaling="linear", factor=0.0), dict(rot_dim=2, scaling="ntk", factor=2.0),
                                dict(rot_dim=64, scaling="yarn", factor=2.0), dict(rot_dim=64, scaling="yarn", factor=0.5, original_length=10),
                                dict(rot_dim=64, scaling="yarn", factor=2.0, original_length=10, low=4.0, high=2.0)])
def test_frequencies_refuse(kw):
    with pytest.raises(ValueError):
        ops.rotary_frequencies(**kw)


def test_long_form_refuses_numbers_past_its_fields():
    """The engine's checks, before its library is called: 32-bit fields take 2^32 + 3 for 3."""
    from f5_tts_amd.engine import F5HipEngine

    eng = F5HipEngine.__new__(F5HipEngine)  # no library, no context: a call that got that far would raise AttributeError
    for kw in (dict(window=1 << 32), dict(window=(1 << 32) + 3), dict(window=(5, 1 << 32)), dict(window=(-(1 << 32), 5)), dict(window=1 << 40),
               dict(window=4, sinks=1 << 32), dict(window=4, sinks=-(1 << 32) + 1), dict(window=1 << 30), dict(window=(-2, 0)), dict(window=4, sinks=1 << 30),
               dict(window=4, rope_scaling="yarn", rope_factor=2.0, rope_original_length=(1 << 64) + 2800)):
        with pytest.raises(ValueError):
            eng.set_long_form(**kw)


@pytest.mark.parametrize("kw", [dict(rot_dim=(1 << 32) + 2), dict(rot_dim=64, scaling="yarn", factor=2.0, original_length=(1 << 64) + 10)])
def test_frequencies_refuse_numbers_past_their_types(kw, monkeypatch):
    monkeypatch.setattr(ops.torch, "tensor", lambda *a, **k: pytest.fail("accepted"))  # (before the list of 2^31 numbers is made)
    if kw["rot_dim"] > 1 << 16:
        monkeypatch.setattr(ops, "load_library", lambda: pytest.fail("accepted"))
    with pytest.raises(ValueError):
        ops.rotary_frequencies(**kw)


@pytest.mark.parametrize("kw", [dict(scaling="linear", factor=1e-310), dict(scaling="ntk", factor=1e-320)])
def test_infinite_frequencies_are_refused(kw):
    with pytest.raises(ValueError, match="infinite"):
        ops.rotary_frequencies(64, **kw)


# ---- refusals: before anything is launched ------------------------------------------------------------------------------------------------
def q4(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def test_rotary_refuses(host):
    f = O.frequencies(64)
    q, k = q4(1, 4, 2, 64), q4(1, 4, 1, 64)
    host.rotary(q, k, f)
    for bad in (dict(q=q[0]), dict(q=q.long()), dict(k=k.float()), dict(k=q4(1, 5, 1, 64)), dict(k=q4(1, 4, 1, 32)), dict(f=f.float()), dict(f=f[None]),
                dict(f=O.frequencies(128)), dict(f=f[:0]), dict(layout="both"), dict(positions=torch.zeros(4)), dict(positions=torch.zeros(5, dtype=torch.int64)),
                dict(positions=torch.zeros(2, 4, dtype=torch.int64)), dict(rot_heads=-2), dict(amplitude=float("inf")), dict(offset=1 << 63),
                dict(out=(q, None)), dict(out=(q, q)), dict(out=(q4(1, 4, 64, 2).transpose(2, 3), k)),
                dict(q=q.expand(3, 4, 2, 64), k=None, out=(q.expand(3, 4, 2, 64), None)), dict(q=q.clone().float().requires_grad_(), k=None)):
        a = dict(q=q, k=k, f=f)
        a.update(bad)
        with pytest.raises(ValueError):
            host.rotary(a.pop("q"), a.pop("k"), a.pop("f"), **a)
    with torch.no_grad():
        host.rotary(q.float().requires_grad_(), None, f)


def test_window_attention_refuses(host):
    q, k, v = q4(2, 3, 4, 64), q4(2, 5, 2, 64), q4(2, 5, 2, 64)
    host.window_attention(q, k, v)
    for bad in (dict(q=q[0]), dict(q=q.double()), dict(k=k.bfloat16()), dict(v=q4(2, 4, 2, 64)), dict(k=q4(1, 5, 2, 64), v=q4(1, 5, 2, 64)),
                dict(k=q4(2, 5, 3, 64), v=q4(2, 5, 3, 64)), dict(q=q4(2, 3, 4, 60), k=q4(2, 5, 2, 60), v=q4(2, 5, 2, 60)),
                dict(q=q4(2, 3, 4, 136), k=q4(2, 5, 2, 136), v=q4(2, 5, 2, 136)), dict(sinks=-1), dict(sinks=1 << 30), dict(window=(1 << 30, 0)),
                dict(window=(1 << 40, 0)), dict(align="middle"), dict(scale=float("nan")), dict(kv_len=torch.zeros(3, dtype=torch.int32)),
                dict(kv_len=torch.zeros(2)), dict(q_len=[1, 2]), dict(out=q4(2, 3, 4, 32)), dict(out=q4(2, 3, 4, 64, dtype=torch.float32)),
                dict(out=q4(2, 3, 4, 66)[..., 1:65]), dict(out=q4(1, 3, 4, 64).expand(2, 3, 4, 64)), dict(q=q4(2, 3, 0, 64)),
                dict(q=q4(2, 3, 4, 0), k=q4(2, 5, 2, 0), v=q4(2, 5, 2, 0)), dict(q=q.float().requires_grad_(), k=k.float(), v=v.float())):
        a = dict(q=q, k=k, v=v)
        a.update(bad)
        with pytest.raises(ValueError):
            host.window_attention(a.pop("q"), a.pop("k"), a.pop("v"), **a)


def test_outputs_that_overlap_are_refused(host):
    f, x = O.frequencies(64), q4(2, 4, 2, 64)
    y = q4(2, 4, 2, 64)
    host.rotary(x, y, f, out=(x, y))
    for out in ((y, x), (x, x), (y, q4(2, 4, 2, 64)), (q4(2, 4, 2, 64), x), (x.view(2, 2, 4, 64).transpose(1, 2), y)):
        with pytest.raises(ValueError, match="own input"):
            host.rotary(x, y, f, out=out)
    for i in range(3):
        qkv = [q4(2, 4, 2, 64) for _ in range(3)]
        with pytest.raises(ValueError, match="no memory"):
            host.window_attention(*qkv, out=qkv[i])


def test_outputs_that_overlap_in_part_are_refused(host):
    f = O.frequencies(64)
    buf = q4(2, 6, 12, 64)  # q | k | v | o, three heads each
    q, k, v, o = (buf[:, :, 3 * i:3 * i + 3] for i in range(4))
    host.rotary(q, k, f, out=(q, k))
    host.rotary(q, k, f, out=(v, o))
    host.window_attention(q, k, v, out=o)
    host.window_attention(q[:, :2], k, v, out=q[:, 2:4])  # rows between
    one_head_on = buf[:, :, 1:4]
    for out in ((one_head_on, v), (v, one_head_on), (v, buf[:, :, 7:10]), (buf[:, :, 5:8], o)):
        with pytest.raises(ValueError, match="own input"):
            host.rotary(q, k, f, out=out)
    with pytest.raises(ValueError, match="own input"):
        host.rotary(buf.flatten()[:6 * 192].view(1, 6, 3, 64), None, f, out=(buf.flatten()[1:6 * 192 + 1].view(1, 6, 3, 64), None))
    for out in (one_head_on, buf[:, :, 2:5], buf[:, :, 8:11], buf.flatten()[8 * 64:8 * 64 + 2 * 6 * 192].view(2, 6, 3, 64)):
        with pytest.raises(ValueError, match="no memory"):
            host.window_attention(q, k, v, out=out)
    lens = buf.view(torch.int32)[0, 0, 11, :2]
    for kw in (dict(kv_len=lens), dict(q_len=lens)):
        with pytest.raises(ValueError, match="lengths"):
            host.window_attention(q, k, v, out=o, **kw)
    wide = torch.zeros(4 * 64, dtype=torch.float64)
    y = wide.view(torch.float32)
    with pytest.raises(ValueError, match="inv_freq"):
        host.rotary(torch.zeros(1, 1, 1, 64), None, wide[:32], out=(y[32:96].view(1, 1, 1, 64), None))
    with pytest.raises(ValueError, match="positions"):
        host.rotary(torch.zeros(2, 4, 1, 64), None, f, positions=y.view(torch.int64)[-8:].view(2, 4), out=(y[:512].view(2, 4, 1, 64), None))
    with pytest.raises(ValueError, match="elements"):
        host.rotary(torch.zeros(2, 4, 1, 64), None, f, out=(y.as_strided((2, 4, 1, 64), (128, 32, 64, 1)), None))
    with pytest.raises(ValueError, match="elements"):
        host.window_attention(q, k, v, out=torch.zeros(2, 6, 3, 64).half().as_strided((2, 6, 3, 64), (64, 128, 64, 1)))


@shim
def test_overlaps_are_found_exactly_on_the_shim(host):
    """Random views of one buffer, the refusal against the sets of their elements."""
    rng, f = random.Random(5), O.frequencies(4)
    said = {True: 0, False: 0}
    for _ in range(3000):
        shape = (rng.randint(1, 3), rng.randint(1, 4), rng.randint(1, 3), 4)
        buf = torch.zeros(700)
        views, cells = [], []
        for _ in range(2):
            st = [rng.choice([0, 1, 2, 3, 4, 5, 8, 12, 13, 16, 24, 36, 48, 49]) if m > 1 else 0 for m in shape[:3]]
            at = rng.choice([0, 4, 12, 17, rng.randint(0, 200)])
            views.append(buf.as_strided(shape, (*st, 1), at))
            cells.append(torch.arange(700).as_strided(shape, (*st, 1), at).flatten().tolist())
        if rng.random() < 0.2:
            views[1], cells[1] = views[0], cells[0]
        (x, y), (a, b) = views, cells
        wrong = len(set(b)) < len(b) or (bool(set(a) & set(b)) and x is not y and not (x.data_ptr() == y.data_ptr() and x.stride() == y.stride()))
        try:
            host.rotary(x, None, f, out=(y, None))
            refused = False
        except ValueError as e:
            refused = True
            assert "output" in str(e), e
        assert refused == wrong, (shape, x.stride(), y.stride(), x.storage_offset(), y.storage_offset())
        said[wrong] += 1
    assert min(said.values()) > 300


def test_scales_that_overflow_are_refused(host):
    x = q4(1, 4, 2, 64)
    for scale in (3e38, -3e38, 2.4e38):  # 2^128 / log2(e) = 2.3587e38
        with pytest.raises(ValueError, match="scale"):
            host.window_attention(x, x, x, scale=scale)
    host.window_attention(x, x, x, scale=2.3e38)


def test_frequencies_that_require_a_gradient_are_refused(host):
    x, f = q4(1, 4, 2, 64), O.frequencies(64).requires_grad_()
    for layout in ("interleaved", "half"):
        with pytest.raises(ValueError, match="gradient"):
            host.rotary(x, None, f, layout=layout)
    with torch.no_grad():
        host.rotary(x, None, f)
    host.rotary(x, None, f.detach())


def test_numbers_that_require_a_gradient_are_refused(host):
    x, f, learned = q4(1, 4, 2, 64), O.frequencies(64), torch.tensor(0.5, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        host.rotary(x, None, f, amplitude=learned)
    with pytest.raises(ValueError, match="gradient"):
        host.window_attention(x, x, x, scale=learned)
    host.rotary(x, None, f, amplitude=learned.detach())
    host.window_attention(x, x, x, scale=learned.detach())


def test_forward_mode_tangents_are_refused(host):
    from torch.autograd import forward_ad as fw

    x, f = q4(1, 4, 2, 64, dtype=torch.float32), O.frequencies(64)
    with fw.dual_level():
        dual, turn = fw.make_dual(x, torch.ones_like(x)), fw.make_dual(f, torch.ones_like(f))
        for args in ((dual, None, f), (x, dual, f), (x, None, turn)):
            with pytest.raises(ValueError, match="tangent"):
                host.rotary(*args)
        with pytest.raises(ValueError, match="tangent"):
            host.rotary(x, None, f, out=(dual, None))
        for i in range(3):
            qkv = [x, x, x]
            qkv[i] = dual
            with pytest.raises(ValueError, match="tangent"):
                host.window_attention(*qkv)
        with pytest.raises(ValueError, match="tangent"):
            host.window_attention(x, x, x, out=fw.make_dual(torch.zeros_like(x), torch.ones_like(x)))
        host.window_attention(x, x, host.rotary(fw.unpack_dual(dual).primal, None, f)[0])


def test_numbers_past_fp32_are_refused(host):
    x = q4(1, 4, 2, 64)
    with pytest.raises(ValueError):
        host.rotary(x, None, O.frequencies(64), amplitude=1e39)
    with pytest.raises(ValueError):
        host.window_attention(x, x, x, scale=1e39)


class RotaryC(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("dtype", "layout", "inverse", "rot_dim", "batch", "tokens", "heads_q", "heads_k", "head_dim", "rot_heads")] + \
        [("amplitude", C.c_float)] + [(n, C.c_void_p) for n in ("q", "k", "q_out", "k_out")] + \
        [(n, C.c_int64 * 3) for n in ("q_stride", "k_stride", "q_out_stride", "k_out_stride")] + \
        [("inv_freq", C.c_void_p), ("positions", C.c_void_p), ("position_stride", C.c_int64), ("first", C.c_int64)]


def rotary_c(**kw):
    """f5hip_rotary_args of 2 x 4 tokens of 2 heads of 64, fp16; the pointers are nobody's memory: for calls that are refused."""
    a = RotaryC(dtype=1, rot_dim=64, batch=2, tokens=4, heads_q=2, head_dim=64, rot_heads=-1, amplitude=1.0, q=1 << 40, q_out=1 << 41, inv_freq=1 << 42)
    a.q_stride[:] = a.q_out_stride[:] = [512, 128, 64]
    for name, x in kw.items():
        if isinstance(x, list):
            getattr(a, name)[:] = x
        else:
            setattr(a, name, x)
    return a


def refusal(lib, a):
    code = lib.f5hip_rotary(C.addressof(a), 0, None)
    return code, lib.f5hip_last_error(None).decode()


def test_rotary_refuses_offsets_past_64_bits(operators_emu_lib):
    """Sizes and strides that are each within their limits, products that are not; nothing is launched."""
    for kw, why in ((dict(tokens=1 << 30, q_stride=[0, 1 << 40, 64]), "span"), (dict(batch=1 << 20, q_out_stride=[1 << 40, 128, 64]), "span"),
                    (dict(batch=1 << 20, positions=1 << 43, position_stride=1 << 40, q_stride=[0, 128, 64]), "positions"),
                    (dict(first=(1 << 63) - 4), "first"), (dict(first=(1 << 63) - 1), "first")):
        code, text = refusal(operators_emu_lib, rotary_c(**kw))
        assert code == 1 and why in text, (kw, text)


def test_rotary_refuses_more_threads_than_it_can_number(operators_emu_lib):
    n, heads = 1 << 23, 32
    big = dict(batch=1, tokens=n, heads_q=heads, inv_freq=1 << 50)
    for odd in (2, 0):  # a pointer that is aligned to one element only: a piece is a pair
        a = rotary_c(q=(1 << 40) + odd, q_out=(1 << 45) + odd, q_stride=[0, heads * 64, 64], q_out_stride=[0, heads * 64, 64], **big)
        if odd:
            code, text = refusal(operators_emu_lib, a)
            assert code == 1 and "pieces" in text
        else:  # 16-byte pieces: 2^30 threads are none too many (device 7 is one too many, so nothing is launched)
            assert operators_emu_lib.f5hip_rotary(C.addressof(a), 7, None) == 1 and b"device" in operators_emu_lib.f5hip_last_error(None)


def test_a_workspace_among_the_tensors_is_refused(operators_emu_lib):
    lib, heads, n, d = operators_emu_lib, 4, 4000, 64
    at = {"q": 1 << 40, "k": 1 << 41, "v": 1 << 42, "out": 1 << 43, "kv_len": 1 << 44, "q_len": 1 << 45}  # nobody's memory: no call is launched
    st = [heads * d, heads * d, d, n * heads * d, heads * d, d, n * heads * d, heads * d, d, heads * d, heads * d, d]

    def pack(work, size):
        return ops._WINDOW.pack(1, 2, 1, n, heads, heads, d, -1, -1, 0, 0, 0.125, *(at[x] for x in ("q", "k", "v", "out")), *st, at["kv_len"], at["q_len"], work, size)

    need = lib.f5hip_window_attention_workspace(pack(0, 0))
    assert need > 0
    ends = {"q": 2 * heads * d * 2, "k": 2 * n * heads * d * 2, "v": 2 * n * heads * d * 2, "out": 2 * heads * d * 2, "kv_len": 8, "q_len": 8}
    for name, base in at.items():
        for work in (base, base + (ends[name] - 1) // 16 * 16, base - need // 16 * 16 + 16):
            assert lib.f5hip_window_attention(pack(work, need), 0, None) == 1 and b"share no memory" in lib.f5hip_last_error(None), (name, work)
        after = base + (ends[name] + 15) // 16 * 16  # (device 7 is one too many, so nothing is launched)
        assert lib.f5hip_window_attention(pack(after, need), 7, None) == 1 and b"device" in lib.f5hip_last_error(None), name


def test_a_library_without_the_operators_is_refused(tmp_path):
    """The operators came without a new ABI version, so their absence has to be said."""
    (tmp_path / "old.c").write_text("int f5hip_abi_version_of_an_old_library(void) { return 10; }\n")
    old = str(tmp_path / "libold.so")
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", old, str(tmp_path / "old.c")], check=True)
    with pytest.raises(binding.F5HipError, match="does not export"):
        binding.load_library(old)


def test_c_entries_refuse_null_and_say_why():
    lib = binding.load_library()
    assert lib.f5hip_rotary(None, 0, None) == 1 and b"null" in lib.f5hip_last_error(None)
    assert lib.f5hip_window_attention(None, 0, None) == 1 and b"null" in lib.f5hip_last_error(None)
    assert lib.f5hip_window_attention_workspace(None) == -1
    a = C.c_double()
    assert lib.f5hip_rotary_frequencies(64, 1e4, 0, 1.0, 0, 0.0, 0.0, None, C.byref(a)) == 1


@pytest.mark.skipif(torch.cuda.is_available(), reason="only meaningful without a GPU")
def test_no_cpu_path():
    with pytest.raises(binding.F5HipError):
        ops.rotary(q4(1, 1, 1, 64), None, O.frequencies(64))
    with pytest.raises(binding.F5HipError):
        ops.window_attention(q4(1, 1, 1, 64), q4(1, 1, 1, 64), q4(1, 1, 1, 64))


def test_empty_calls(host):
    f = O.frequencies(64)
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64)):
        a, b = host.rotary(q4(*shape), q4(*shape), f)
        assert a.shape == b.shape == shape
        assert host.window_attention(q4(*shape), q4(shape[0], 5, 2, 64), q4(shape[0], 5, 2, 64)).shape == shape


# ---- the kernels' source on the host shim ---------------------------------------------------------------------------------------------------
@shim
@pytest.mark.parametrize("name", sorted(O.ROTARY))
def test_rotary_on_the_shim(host, name):
    O.check_rotary(host, same, O.ROTARY[name])


@shim
def test_rotary_amplitude_positions_views_and_in_place_on_the_shim(host):
    g = torch.Generator().manual_seed(1)
    fused = torch.randn(2, 7, 6, 64, generator=g).half()
    q, k, f = fused[:, :, :3], fused[:, :, 3:5], O.frequencies(48)
    at = torch.randint(-1000, 200000, (2, 7), generator=g)
    want = [O.rotary(x, f, at, amplitude=1.2, half=True) for x in (q, k)]
    got = host.rotary(q, k, f, amplitude=1.2, positions=at, layout="half")
    for y, (ref, tol) in zip(got, want):
        assert O.over(y, ref, tol) <= 1
    before = fused.clone()
    host.rotary(q, k, f, amplitude=1.2, positions=at, layout="half", out=(q, k))  # in place, in the fused buffer
    assert torch.equal(q, got[0]) and torch.equal(k, got[1]) and torch.equal(fused[:, :, 5:], before[:, :, 5:])
    shared = host.rotary(before[:, :, :3], None, f, positions=at[0])[0]  # one row of positions for all sequences
    assert torch.equal(shared, host.rotary(before[:, :, :3], None, f, positions=at[:1].expand(2, 7))[0])
    odd = torch.randn(2 * 3 * 2 * 64 + 1, generator=g).half()[1:].view(2, 3, 2, 64)  # not aligned to more than an element
    ref, tol = O.rotary(odd, f, torch.arange(3))
    assert O.over(host.rotary(odd, None, f)[0], ref, tol) <= 1
    turned = host.rotary(before[:, :, :1].expand(2, 7, 3, 64), None, f)[0]  # a broadcast input
    assert torch.equal(turned[:, :, 0], turned[:, :, 2])


@shim
@pytest.mark.parametrize("name", sorted(O.ATTENTION))
def test_window_attention_on_the_shim(host, name):
    O.check_attention(host, same, O.ATTENTION[name])


@shim
def test_window_attention_ignores_what_nobody_sees_on_the_shim(host):
    check_unseen(host, same)


@shim
def test_window_attention_of_huge_scores_on_the_shim(host):
    O.check_huge_scores(host, same)


@shim
def test_lengths_are_clamped_whatever_their_type_on_the_shim(host):
    q, k, v, kw = O.attention_inputs(O.ATTENTION["chunk"])
    kw.pop("kv_len"), kw.pop("q_len")
    want = host.window_attention(q, k, v, **kw)
    tq, tk = q.shape[1], k.shape[1]
    for lens in ([2 ** 63 - 1, 2 ** 32 + 1], [2 ** 31, 2 ** 32], [tk, tk + 1]):  # all of them, in 64 bits
        assert torch.equal(host.window_attention(q, k, v, kv_len=torch.tensor(lens), q_len=torch.tensor(lens), **kw), want)
    for low in (-1, -2 ** 32 + tq, -2 ** 63):  # none
        n = torch.tensor([tq, low])
        got = host.window_attention(q, k, v, q_len=n, **kw)
        assert torch.equal(got[0], want[0]) and (got[1] == 0).all()
        got = host.window_attention(q, k, v, kv_len=torch.tensor([tk, low]), **kw)
        assert torch.equal(got[0], want[0]) and (got[1] == 0).all()


@shim
def test_writes_are_noticed_by_autograd_on_the_shim(host):
    f, x = O.frequencies(64), torch.randn(2, 4, 2, 64, generator=torch.Generator().manual_seed(2))
    calls = [lambda y: host.rotary(y, None, f, out=(y, None)), lambda y: host.rotary(x, x, f, out=(torch.empty_like(x), y)),
             lambda y: host.window_attention(x, x, x, out=y), lambda y: host.rotary(x, y[:, :, :1], f, out=(torch.empty_like(x), y[:, :, :1]))]
    for call in calls:
        y, w = x.clone(), torch.ones_like(x, requires_grad=True)
        loss = (w * y).sum()  # saves y
        call(y)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():  # such tensors count no versions
        y = x.clone()
        host.rotary(y, y.clone(), f, out=(y, torch.empty_like(y)))
        host.window_attention(y, y, y, out=torch.empty_like(y))


@shim
@pytest.mark.parametrize("name", sorted(K.MORE_ATTENTION))
def test_more_window_attention_on_the_shim(host, name):
    O.check_attention(host, same, K.MORE_ATTENTION[name], seed=8)


@shim
def test_window_attention_of_nan_keys_on_the_shim(host):
    K.check_nan_keys(host, same)


@shim
def test_rotary_of_far_positions_on_the_shim(host):
    assert abs(float(K.TURN) * 2 * math.pi - 1) < 2.0 ** -51
    K.check_far_positions(host, same)


@shim
def test_window_attention_of_large_values_on_the_shim(host):
    K.check_large_values(host, same)


@shim
def test_axes_of_one_element_carry_any_stride_on_the_shim(host):
    x = torch.randn(128, generator=torch.Generator().manual_seed(4)).half()
    plain, odd = x.view(1, 1, 2, 64), x.as_strided((1, 1, 2, 64), (7, (1 << 40) + 3, 64, 1))
    f = O.frequencies(64)
    assert torch.equal(host.rotary(odd, odd, f, offset=3)[1], host.rotary(plain, None, f, offset=3)[0])
    assert torch.equal(host.window_attention(odd, odd, odd), host.window_attention(plain, plain, plain))
    out, one = torch.zeros(64).half().as_strided((1, 1, 1, 64), (0, 0, 3, 1)), plain[:, :, :1]
    assert torch.equal(host.window_attention(one, one, one, out=out), host.window_attention(one, one, one))
    fits = x.as_strided((1, 1, 2, 64), (7, 3, 64, 1))
    assert ops._rows(fits)[0] is fits  # not copied


@shim
def test_window_attention_of_a_nan_on_the_shim(host):
    O.check_seen_nan(host, same)


def check_unseen(ops_, to):
    """Keys and values behind the last key, and in front of every window but no sink, may hold NaN and infinities."""
    for name in ("token_grouped", "chunk", "token_fp32", "ragged"):
        case = O.ATTENTION[name]
        q, k, v, kw = O.attention_inputs(case)
        tq, tk = q.shape[1], k.shape[1]
        for i in range(q.shape[0]):
            n = tk if kw["kv_len"] is None else int(kw["kv_len"][i])
            k[i, n:], v[i, n:] = math.nan, math.inf
            if kw["align"] == "end":
                low = max(0, n - tq - kw["window"][0])
                k[i, kw["sinks"]:low], v[i, kw["sinks"]:low] = math.inf, math.nan
        ref, tol, rows = O.attention(q, k, v, **kw)
        out = ops_.window_attention(to(q), to(k), to(v), **{x: to(y) if isinstance(y, torch.Tensor) else y for x, y in kw.items()})
        assert O.over(out, ref, tol) <= 1
