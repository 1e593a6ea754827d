"""Operators with entry points of their own: rotary positions and sliding-window attention on the caller's tensors.

They are what the sampler runs in its blocks after ``F5HipEngine.set_long_form`` (``engine.py``), for programs that bring their own layers:
``[batch, tokens, heads, head_dim]`` tensors with any strides of the first three axes (columns of a fused q|k|v buffer, views of a cache), in
fp32, fp16 or bf16, on the current stream of their device.  The reference calls ``apply_rotary_pos_emb`` and
``F.scaled_dot_product_attention`` in these places (``src/f5_tts/model/modules.py:498-520``).  Nothing is kept between calls: outputs and
workspaces come from torch's allocator on the calling stream, so calls can be captured into graphs and run side by side.  Inference only:
an input that requires a gradient or carries a tangent is refused.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad as _forward_ad

from .binding import ROPE_SCALINGS, F5HipError, check, load_library

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # F5HIP_T_*
_LAYOUTS = {"interleaved": 0, "half": 1}                          # F5HIP_ROTARY_*
_ALIGN = {"start": 0, "end": 1}
_ROTARY = struct.Struct("@10if4P12qPP2q")   # f5hip_rotary_args
_WINDOW = struct.Struct("@11if4P12q3Pq")    # f5hip_window_attention_args


# The calls below take about as long on the host as the small launches do on the GPU: each check is one comparison where it passes.
def _device(t: torch.Tensor) -> Tuple[int, int]:
    """(device ordinal, current stream) of a GPU tensor."""
    if not t.is_cuda:
        raise F5HipError("the operators need tensors on a HIP device (torch device type 'cuda'); there is no CPU path")
    index = t.get_device()
    return index, torch._C._cuda_getCurrentRawStream(index)  # torch.cuda.current_stream(device).cuda_stream without the Python objects (2 us)


def _tensor(name: str, t: torch.Tensor, dtype: Optional[torch.dtype] = None, device: Optional[torch.device] = None) -> None:
    if not isinstance(t, torch.Tensor) or t.dim() != 4:
        raise ValueError(f"{name}: a [batch, tokens, heads, head_dim] tensor is expected")
    if dtype is None:
        if t.dtype not in _TYPES:
            raise ValueError(f"{name}: {t.dtype} is not one of float32, float16, bfloat16")
    elif t.dtype != dtype or t.device != device:
        raise ValueError(f"{name}: {t.dtype} on {t.device}, the first tensor is {dtype} on {device}")
    if t.requires_grad or _forward_ad._current_level >= 0:
        _inference(name, t)


def _inference(name: str, t: torch.Tensor) -> None:
    """Refuses what would lose a derivative.  Called where a tensor requires a gradient or a dual level is open (not -1)."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: the operators are for inference (use torch.no_grad())")
    if _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} carries a tangent of forward-mode differentiation: the operators are for inference (use its primal)")


def _lengths(name: str, t: Optional[torch.Tensor], like: torch.Tensor, most: int) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64) or t.shape != like.shape[:1] or t.device != like.device:
        raise ValueError(f"{name}: an int32 or int64 tensor of [batch] on {like.device} is expected")
    if t.dtype == torch.int64:
        t = t.clamp(0, most).to(torch.int32)  # (the kernels clamp 32-bit lengths; narrowed first, 2^32 + 1 would be 1)
    return t.contiguous()


# a tensor, or an iterable of them, was written behind torch's back: an operation that saved it for its backward pass has to notice
_written = torch.autograd.graph.increment_version


def _pack(layout: struct.Struct, fields) -> bytes:
    try:
        return layout.pack(*fields)
    except struct.error as e:  # a size or an option that does not fit its field
        raise ValueError(f"argument out of range: {e}") from None


def rotary_frequencies(rot_dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0, original_length: int = 0,
                       low: float = 0.0, high: float = 0.0, device=None) -> Tuple[torch.Tensor, float]:
    """``(inv_freq, amplitude)`` for :func:`rotary`: ``rot_dim / 2`` frequencies in 64 bits (on ``device``), scaled for contexts ``factor``
    times as long as trained — ``"linear"`` (positions interpolated), ``"ntk"`` (the base changed) or ``"yarn"`` (by parts: frequencies that turn
    less than ``low`` (1) times over ``original_length`` positions are divided, those above ``high`` (32) kept, mixed between them)."""
    if scaling not in ROPE_SCALINGS:
        raise ValueError(f"scaling {scaling!r}: one of None, 'linear', 'ntk', 'yarn' is expected")
    if not 0 < rot_dim <= 1 << 16 or not 0 <= original_length < 1 << 63:  # (the C arguments would take larger ones modulo 2^32 and 2^64)
        raise ValueError(f"rot_dim {rot_dim} must be in [2, 65536], original_length {original_length} in [0, 2^63)")
    out, amplitude = (C.c_double * max(1, rot_dim // 2))(), C.c_double()
    lib = load_library()
    check(lib, None, lib.f5hip_rotary_frequencies(rot_dim, base, ROPE_SCALINGS[scaling], factor, original_length, low, high, out, C.byref(amplitude)))
    return torch.tensor(list(out), dtype=torch.float64, device=device), amplitude.value


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], inv_freq: torch.Tensor, *, amplitude: float = 1.0, positions: Optional[torch.Tensor] = None,
           offset: int = 0, layout: str = "interleaved", rot_heads: Optional[int] = None, inverse: bool = False, out=None):
    """Rotate the pairs of q's and k's columns by their positions' angles, both in one launch; returns ``(q', k')`` (``k`` may be None).

    ``inv_freq``: float64 ``[R / 2]`` on the device (:func:`rotary_frequencies`); the first ``R`` columns of a head rotate, the others are
    copied.  ``layout``: pairs are columns ``(2i, 2i + 1)`` ("interleaved") or ``(i, i + R / 2)`` ("half").  ``positions``: int64
    ``[batch, tokens]`` or ``[tokens]``; without them token t stands at ``offset + t``.  ``rot_heads``: only the first so many heads of q and of
    k rotate (the reference's ``pe_attn_head``).  ``inverse`` turns back (with amplitude 1 the inverse; in any case the operator's gradient).
    ``out``: ``(q', k')`` to write to — the inputs themselves, or tensors that share no element with them (other columns of one buffer do not)."""
    _tensor("q", q)
    dtype, where, shape = q.dtype, q.device, q.shape
    if layout not in _LAYOUTS:
        raise ValueError(f"layout {layout!r}: 'interleaved' or 'half' is expected")
    if not isinstance(inv_freq, torch.Tensor) or inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or inv_freq.device != where:
        raise ValueError(f"inv_freq: a float64 vector on {where} is expected (rotary_frequencies)")
    if inv_freq.requires_grad or _forward_ad._current_level >= 0:
        _inference("inv_freq", inv_freq)
    if type(amplitude) is not float and isinstance(amplitude, torch.Tensor):
        _inference("amplitude", amplitude)
    inv_freq = inv_freq.contiguous()
    b, n, h, d = shape
    hk = 0
    if k is not None:
        _tensor("k", k, dtype, where)
        kshape = k.shape
        hk = kshape[2]
        if kshape[0] != b or kshape[1] != n or kshape[3] != d or hk == 0:
            raise ValueError(f"k is {tuple(kshape)}, q {tuple(shape)}: batch, tokens and head_dim must agree")
    if out is None:
        if q.stride(3) != 1:
            q = q.contiguous()
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        k_out = None
        if k is not None:
            if k.stride(3) != 1:
                k = k.contiguous()
            k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    else:
        q_out, k_out = out
        for name, x, y in (("q", q, q_out), ("k", k, k_out)):
            if (x is None) != (y is None):
                raise ValueError(f"out: one tensor for q and one for k is expected, None for a {name} that is None")
            if x is None:
                continue
            _tensor(f"out for {name}", y, dtype, where)
            if y.shape != x.shape:
                raise ValueError(f"out for {name} is {tuple(y.shape)}, {name} {tuple(x.shape)}")
            if x.stride(3) != 1 or y.stride(3) != 1:
                raise ValueError(f"{name}: with out the last axis of input and output must be contiguous")
    step = 0
    if positions is not None:
        if not isinstance(positions, torch.Tensor) or positions.dtype != torch.int64 or positions.device != where or \
                tuple(positions.shape) not in ((n,), (1, n), (b, n)):
            raise ValueError(f"positions: int64 of [tokens] or [batch, tokens] on {where} is expected")
        positions = positions.contiguous()
        step = n if positions.dim() == 2 and positions.shape[0] > 1 else 0
    device, stream = _device(q)
    zero = (0, 0, 0)
    args = _pack(_ROTARY, (_TYPES[dtype], _LAYOUTS[layout], 1 if inverse else 0, 2 * inv_freq.shape[0], b, n, h, hk, d,
                           -1 if rot_heads is None else rot_heads, amplitude, q.data_ptr(), 0 if k is None else k.data_ptr(), q_out.data_ptr(),
                           0 if k is None else k_out.data_ptr(), *q.stride()[:3], *(zero if k is None else k.stride()[:3]), *q_out.stride()[:3],
                           *(zero if k is None else k_out.stride()[:3]), inv_freq.data_ptr(), 0 if positions is None else positions.data_ptr(), step, offset))
    lib = load_library()
    status = lib.f5hip_rotary(args, device, stream)
    if status:
        check(lib, None, status)
    if out is not None:
        _written(q_out if k is None else (q_out, k_out))
    return q_out, k_out


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, Tuple[int, int, int, int]]:
    """The tensor, or a copy, with 16-byte aligned rows, and its strides."""
    st = t.stride()
    if st[3] == 1:
        if ((st[0] | st[1] | st[2]) * t.element_size() | t.data_ptr()) % 16 == 0:
            return t, st
        if t.data_ptr() % 16 == 0 and all(m <= 1 or x * t.element_size() % 16 == 0 for x, m in zip(st[:3], t.shape)):
            return t, st  # an axis of one element may carry any stride
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride()


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: Tuple[int, int] = (-1, -1), sinks: int = 0,
                     kv_len: Optional[torch.Tensor] = None, q_len: Optional[torch.Tensor] = None, align: str = "start",
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of q ``[batch, q_tokens, heads, D]`` over k, v ``[batch, kv_tokens, kv_heads, D]`` through a sliding window; like q.

    Query i stands at ``p = i`` (``align="start"``) or at the end of the keys, ``p = kv_len - q_len + i`` (``align="end"``: new tokens, one or
    many, over a cache that holds theirs as its last).  With ``window = (left, right)`` it sees the keys ``p - left <= j <= p + right`` (negative:
    no bound on that side; ``right = 0``: causal) and, of the first ``sinks`` keys, all that ``right`` allows.  A query that sees no key gives
    zeros.  ``kv_len``, ``q_len``: valid keys and queries of each sequence; output rows behind ``q_len`` are zero, or left as they were in
    ``out``.  ``scale``: 1 / sqrt(D) by default.  D: a multiple of 8 (fp32: 4) up to 128.  Keys and values that no query sees may hold
    anything, a value that some query sees has to be finite for the others' sake; tensors whose rows are not aligned to 16 bytes are copied first.
    Scaled scores have to stay below 2^22 in magnitude (past some 2^28 in fp16 and 2^32 in the others the result is NaN), and 16 |v| times the
    keys of a query below 2^128.  In fp32 an infinity that a query sees gives NaN; in fp16 and bf16 a key that scores -inf has no weight.  ``out``
    shares no element with q, k and v."""
    _tensor("q", q)
    dtype, where, shape = q.dtype, q.device, q.shape
    _tensor("k", k, dtype, where)
    _tensor("v", v, dtype, where)
    b, n, h, d = shape
    kshape = k.shape
    if kshape != v.shape or kshape[0] != b or kshape[3] != d:
        raise ValueError(f"q {tuple(shape)}, k {tuple(kshape)}, v {tuple(v.shape)}: batch and head_dim must agree, k and v in all axes")
    if d == 0 or h == 0 or kshape[2] == 0:
        raise ValueError(f"q {tuple(shape)}, k {tuple(kshape)}: heads and head_dim must be positive")
    if scale is not None and isinstance(scale, torch.Tensor):
        _inference("scale", scale)
    if align not in _ALIGN:
        raise ValueError(f"align {align!r}: 'start' or 'end' is expected")
    kv_len, q_len = _lengths("kv_len", kv_len, q, kshape[1]), _lengths("q_len", q_len, q, n)
    left, right = window
    given = out
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format) if q_len is None else torch.zeros(shape, dtype=dtype, device=where)
    else:
        _tensor("out", out, dtype, where)
        if out.shape != shape:
            raise ValueError(f"out is {tuple(out.shape)}, q {tuple(shape)}")
        if out.stride(3) != 1:
            raise ValueError("out: the last axis must be contiguous")
    q, qs = _rows(q)
    k, ks = _rows(k)
    v, vs = _rows(v)
    device, stream = _device(q)
    lib = load_library()
    fields = [_TYPES[dtype], b, n, kshape[1], h, kshape[2], d, left, right, sinks, _ALIGN[align], d ** -0.5 if scale is None else scale,
              q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), *qs[:3], *ks[:3], *vs[:3], *out.stride()[:3],
              0 if kv_len is None else kv_len.data_ptr(), 0 if q_len is None else q_len.data_ptr(), 0, 0]
    args = _pack(_WINDOW, fields)
    need = lib.f5hip_window_attention_workspace(args)
    if need < 0:
        check(lib, None, 1)
    if need:
        work = torch.empty(need, dtype=torch.uint8, device=where)
        fields[-2:] = [work.data_ptr(), need]
        args = _pack(_WINDOW, fields)
    status = lib.f5hip_window_attention(args, device, stream)
    if status:
        check(lib, None, status)
    if given is not None:
        _written(out)
    return out
