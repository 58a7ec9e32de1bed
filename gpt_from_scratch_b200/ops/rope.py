"""Rotary position embedding.

:func:`apply_rope` rotates interleaved pairs of the whole head (csrc/elementwise.cu: rope_kernel);
:func:`rotary` (csrc/rotary.cu) is the general form: pairs side by side or half apart, part of the head,
a position for every token; :func:`rope_tables` makes its tables, scaled for longer contexts if need be.

``x'[2i] = x[2i] cos - x[2i+1] sin``, ``x'[2i+1] = x[2i] sin + x[2i+1] cos``; the backward
is the inverse rotation. Same math as the reference's Triton kernel
(core/rope_triton.py:112-133), but q and k are rotated by one launch, in place,
inside the packed qkv buffer. cos/sin are fp32 ``[S, D/2]`` tables.
"""
from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass

import torch

from . import _lib


def rope_reference(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x: ``[S, B, nh, D]``; cos, sin: ``[S, D/2]``."""
    S = x.shape[0]
    c = cos[:S].float()[:, None, None, :]
    s = sin[:S].float()[:, None, None, :]
    xe = x[..., 0::2].float()
    xo = x[..., 1::2].float()
    out = torch.stack((xe * c - xo * s, xe * s + xo * c), dim=-1).flatten(-2)
    return out.to(x.dtype)


def rope_inplace_native(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, S: int, B: int, nh: int, D: int,
                        parts: int, token_stride: int, backward: bool, s_offset: int = 0) -> None:
    assert cos.dtype == torch.float32 and sin.dtype == torch.float32 and cos.is_contiguous() and sin.is_contiguous()
    assert cos.shape[0] >= S + s_offset and cos.shape[1] == D // 2
    rc = _lib.lib().gfs_rope(x.data_ptr(), cos.data_ptr(), sin.data_ptr(), S, B, nh, D, parts, token_stride,
                             1 if backward else 0, s_offset, _lib.stream_ptr())
    _lib.check(rc, "gfs_rope")


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, cos, sin):
        S, B, nh, D = x.shape
        out = x.contiguous().clone()
        rope_inplace_native(out, cos, sin, S, B, nh, D, 1, nh * D, False)
        ctx.save_for_backward(cos, sin)
        return out

    @staticmethod
    def backward(ctx, g):
        cos, sin = ctx.saved_tensors
        S, B, nh, D = g.shape
        dx = g.contiguous().clone()
        rope_inplace_native(dx, cos, sin, S, B, nh, D, 1, nh * D, True)
        return dx, None, None


def apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Rotate ``x [S, B, nh, D]`` (reference API: core/rope_triton.py:144)."""
    if x.is_cuda and x.dtype == torch.bfloat16 and x.shape[-1] % 8 == 0:
        return _Rope.apply(x, cos.float().contiguous(), sin.float().contiguous())
    return rope_reference(x, cos, sin)


def apply_rope_qk(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor):
    """Rotate q and k (reference API: core/rope_triton.py:147-148)."""
    return apply_rope(q, cos, sin), apply_rope(k, cos, sin)


# ---------------------------------------------------------------------------------------------- general form
@dataclass(frozen=True)
class RopeScaling:
    """How the angles of :func:`rope_tables` change for contexts ``factor`` times longer than trained on.

    ``kind``: ``"linear"`` divides every position by ``factor``; ``"ntk"`` raises the base to ``base *
    factor^(R / (R - 2))``, which divides the lowest frequency by ``factor`` and leaves the highest;
    ``"by_parts"`` divides the frequencies that turn fewer than ``low`` times in ``original_length`` tokens,
    leaves those that turn more than ``high`` times, and blends in between. cos and sin are multiplied by
    ``magnitude`` (``None``: ``0.1 ln(factor) + 1``)."""
    kind: str
    factor: float
    original_length: int = 0
    low: float = 1.0
    high: float = 32.0
    magnitude: float | None = 1.0

    def __post_init__(self):
        if self.kind not in ("linear", "ntk", "by_parts"):
            raise ValueError(f"RopeScaling: unknown kind {self.kind!r} (linear, ntk and by_parts are known)")
        if not (self.factor > 0.0 and math.isfinite(self.factor)):
            raise ValueError(f"RopeScaling: factor {self.factor} is not positive")
        if self.kind == "by_parts" and not (self.original_length > 0 and self.low < self.high):
            raise ValueError("RopeScaling: by_parts needs original_length > 0 and low < high")


def rope_tables(length: int, rotary_dim: int, base: float = 10000.0, scaling: RopeScaling | None = None,
                device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """cos and sin, fp32 ``[length, rotary_dim / 2]``: row p holds the angles ``p base^(-2i / rotary_dim)``.

    Angles are 64-bit: those of far positions are large, and 32 bits would leave them few digits."""
    if length < 0 or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rope_tables: length {length} or rotary_dim {rotary_dim} (has to be even) does not do")
    at = torch.arange(length, dtype=torch.float64, device=device)
    exponent = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim
    magnitude = 1.0
    if scaling is not None:
        magnitude = scaling.magnitude if scaling.magnitude is not None else 0.1 * math.log(scaling.factor) + 1.0
        if scaling.kind == "ntk":
            if rotary_dim <= 2:
                raise ValueError("rope_tables: ntk scaling needs rotary_dim > 2")
            base = base * scaling.factor ** (rotary_dim / (rotary_dim - 2))
    freq = base ** -exponent
    if scaling is not None and scaling.kind == "linear":
        freq = freq / scaling.factor
    elif scaling is not None and scaling.kind == "by_parts":
        turns = scaling.original_length * freq / (2.0 * math.pi)
        keep = ((turns - scaling.low) / (scaling.high - scaling.low)).clamp(0.0, 1.0)
        freq = freq * keep + freq / scaling.factor * (1.0 - keep)
    angles = torch.outer(at, freq)
    return (angles.cos() * magnitude).float(), (angles.sin() * magnitude).float()


NATIVE_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_HEAD_DIM = 256


@functools.lru_cache(maxsize=1024)
def stride_array(*strides: tuple[int, ...]):
    """ctypes array of the first three element strides of each tensor."""
    return (ctypes.c_longlong * (3 * len(strides)))(*(n for st in strides for n in st[:3]))


def rows_of(t: torch.Tensor) -> torch.Tensor:
    """``t`` if its last dimension is contiguous, else a copy that is."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def check_tables(what: str, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None,
                 S: int, B: int, D: int) -> int:
    """Checks the arguments that all rotations share; returns the number of rotated dimensions."""
    table_type = torch.float64 if cos.dtype == x.dtype == torch.float64 else torch.float32
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != table_type or sin.dtype != table_type:
        raise ValueError(f"{what}: cos and sin have to be fp32 tables of one shape [positions, rotary_dim / 2]")
    R = 2 * cos.shape[1]
    if not 0 < R <= D:
        raise ValueError(f"{what}: tables for {R} dimensions do not fit a head of {D}")
    if positions is None:
        if cos.shape[0] < S:
            raise ValueError(f"{what}: tables of {cos.shape[0]} positions are too short for {S} tokens")
    else:
        if positions.shape != (B, S) or positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{what}: positions have to be int32 or int64 of shape [batch, sequence] = [{B}, {S}]")
        if cos.shape[0] == 0 and positions.numel() > 0:
            raise ValueError(f"{what}: the tables are empty")
    for t in (cos, sin, positions):
        if t is not None and t.device != x.device:
            raise ValueError(f"{what}: tables and positions have to be on {x.device}")
    if x.is_cuda:
        if x.dtype not in NATIVE_TYPES:
            raise ValueError(f"{what}: no native kernel for {x.dtype} (bfloat16, float16 and float32 have one)")
        if D > MAX_HEAD_DIM:
            raise ValueError(f"{what}: no native kernel for heads of {D} dimensions (up to {MAX_HEAD_DIM})")
    return R


def rotary_reference(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None = None,
                     interleaved: bool = True) -> torch.Tensor:
    """:func:`rotary` in torch operations: fp32 (64 bits for 64-bit inputs), rounded once."""
    S, R = x.shape[0], 2 * cos.shape[1]
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    if positions is None:
        c, s = cos[:S, None, None], sin[:S, None, None]
    else:
        if positions.numel() and not x.is_cuda and not 0 <= int(positions.min()) <= int(positions.max()) < cos.shape[0]:
            raise ValueError("rotary: a position lies outside of the tables")
        at = positions.t().long()
        c, s = cos[at].unsqueeze(2), sin[at].unsqueeze(2)
    c, s = c.to(wide), s.to(wide)
    head, tail = x[..., :R].to(wide), x[..., R:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        out = torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)
    else:
        a, b = head.chunk(2, dim=-1)
        out = torch.cat((a * c - b * s, a * s + b * c), dim=-1)
    return torch.cat((out.to(x.dtype), tail), dim=-1)


def _rotary_native(x, cos, sin, positions, interleaved: bool, inverse: bool) -> torch.Tensor:
    S, B, nh, D = x.shape
    x = rows_of(x)
    y = torch.empty((S, B, nh, D), dtype=x.dtype, device=x.device)
    with _lib.on_device(x), _lib.nvtx("rotary"):
        rc = _lib.lib().gfs_rotary(x.data_ptr(), y.data_ptr(), stride_array(x.stride(), y.stride()), cos.data_ptr(),
                                   sin.data_ptr(), _lib.ptr(positions),
                                   positions is not None and positions.dtype == torch.int64, cos.shape[0], S, B, nh, D,
                                   2 * cos.shape[1], not interleaved, inverse, NATIVE_TYPES[x.dtype], _lib.stream_ptr())
    _lib.check(rc, "gfs_rotary")
    return y


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, cos, sin, positions, interleaved):
        ctx.save_for_backward(cos, sin, positions)
        ctx.interleaved = interleaved
        ctx.traced = torch._C._is_tracing()
        return _rotary_native(x, cos, sin, positions, interleaved, False)

    @staticmethod
    @_lib.first_order
    def backward(ctx, dy):
        cos, sin, positions = ctx.saved_tensors
        return _rotary_native(dy, cos, sin, positions, ctx.interleaved, True), None, None, None, None


def rotary(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None = None,
           interleaved: bool = True) -> torch.Tensor:
    """Rotate the first ``R`` dimensions of every head of ``x [S, B, heads, D]``; the others stay.

    ``cos``, ``sin``: fp32 ``[n, R / 2]`` tables (:func:`rope_tables`), constants for autograd. Token ``(s, b)`` takes
    row ``s``, or ``positions[b, s]`` (int32 or int64 ``[B, S]``): documents packed into a sequence, tokens far
    into a context. ``interleaved``: pairs ``(2i, 2i + 1)`` as in :func:`apply_rope`, else ``(i, i + R / 2)``. ``x`` may have
    any strides; the result is a new contiguous tensor of its type. On CUDA: bfloat16, float16 or float32 and D up to
    256, no forward-mode derivatives; a position outside of the tables is reported by ``_lib.raise_on_status()`` (on the CPU:
    ValueError).
    """
    if x.dim() != 4:
        raise ValueError(f"rotary: x of shape {tuple(x.shape)} is not [S, B, heads, D]")
    S, B, _, D = x.shape
    check_tables("rotary", x, cos, sin, positions, S, B, D)
    if x.is_cuda:
        args = (x, cos.contiguous(), sin.contiguous(), None if positions is None else positions.contiguous(), interleaved)
        return _rotary_native(*args, False) if _lib.bare(x) else _Rotary.apply(*args)
    return rotary_reference(x, cos, sin, positions, interleaved)
