"""Norms of queries and keys, head by head, with the position rotation in the same pass (csrc/rotary.cu).

From the packed projection ``[S, B, (heads + 2 kv_heads) * D]`` to q and k: ``x / sqrt(mean(x^2) + eps) * w`` over the D
dimensions of every head (one weight for all heads of q, one for all of k), then the rotation of
:func:`~gpt_from_scratch_b200.ops.rope.rotary`. fp32 throughout, rounded once; every element is read and written
once, in the backward too, which recomputes the norm and writes the gradient of the whole projection.
"""
from __future__ import annotations

import torch

from . import _lib
from .rope import NATIVE_TYPES, check_tables, rotary_reference, rows_of, stride_array


def qk_norm_rope_reference(qkv, q_weight, k_weight, cos, sin, num_heads, num_kv_heads, eps=1e-5, positions=None,
                           interleaved=True):
    """The operator in torch operations: fp32 (64 bits for 64-bit inputs), rounded once."""
    wide = torch.float64 if qkv.dtype == torch.float64 else torch.float32
    heads = qkv.unflatten(-1, (num_heads + 2 * num_kv_heads, -1))
    q, k, v = heads.split([num_heads, num_kv_heads, num_kv_heads], dim=2)

    def one(x, w):
        x = x.to(wide)
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.to(wide)
        return rotary_reference(x, cos, sin, positions, interleaved).to(qkv.dtype)
    return one(q, q_weight), one(k, k_weight), v


def _forward(x, q_weight, k_weight, cos, sin, n1, n2, eps, positions, interleaved):
    S, B, W = x.shape
    D = W // (n1 + 2 * n2)
    q = torch.empty((S, B, n1, D), dtype=x.dtype, device=x.device)
    k = torch.empty((S, B, n2, D), dtype=x.dtype, device=x.device)
    ss, bs, _ = x.stride()
    with _lib.on_device(x), _lib.nvtx("qk_norm_rope"):
        rc = _lib.lib().gfs_qk_norm_rope_fwd(
            x.data_ptr(), stride_array((ss, bs, D)), _lib.ptr(q_weight), _lib.ptr(k_weight), q.data_ptr(), k.data_ptr(),
            cos.data_ptr(), sin.data_ptr(), _lib.ptr(positions), positions is not None and positions.dtype == torch.int64,
            cos.shape[0], S, B, n1, n2, D, 2 * cos.shape[1], not interleaved, eps, NATIVE_TYPES[x.dtype],
            _lib.stream_ptr())
    _lib.check(rc, "gfs_qk_norm_rope_fwd")
    return q, k, x.as_strided((S, B, n2, D), (ss, bs, D, 1), x.storage_offset() + (n1 + n2) * D)


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, q_weight, k_weight, cos, sin, n1, n2, eps, positions, interleaved):
        ctx.save_for_backward(qkv, q_weight, k_weight, cos, sin, positions)
        ctx.args = (n1, n2, eps, interleaved)
        ctx.traced = torch._C._is_tracing()
        return _forward(qkv, q_weight, k_weight, cos, sin, n1, n2, eps, positions, interleaved)

    @staticmethod
    @_lib.first_order
    def backward(ctx, dq, dk, dv):
        qkv, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        n1, n2, eps, interleaved = ctx.args
        S, B, W = qkv.shape
        D = W // (n1 + 2 * n2)
        lib = _lib.lib()
        dq, dk, dv = rows_of(dq), rows_of(dk), rows_of(dv)
        dqkv = torch.empty((S, B, W), dtype=qkv.dtype, device=qkv.device)
        if qkv.numel() == 0:
            return dqkv, *(None if w is None else torch.zeros_like(w) for w in (q_weight, k_weight)), *[None] * 7
        dw1 = dw2 = scratch = None
        ss, bs, _ = qkv.stride()
        with _lib.on_device(qkv), _lib.nvtx("qk_norm_rope_bwd"):
            if q_weight is not None:
                dw1, dw2 = torch.empty_like(q_weight), torch.empty_like(k_weight)
                scratch = torch.empty(lib.gfs_qk_norm_rope_scratch(D), dtype=torch.float32, device=qkv.device)
            st = stride_array((ss, bs, D), dq.stride(), dk.stride(), dv.stride(), (B * W, W, D))
            rc = lib.gfs_qk_norm_rope_bwd(
                qkv.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dqkv.data_ptr(), st, _lib.ptr(q_weight),
                _lib.ptr(k_weight), _lib.ptr(dw1), _lib.ptr(dw2), _lib.ptr(scratch), cos.data_ptr(), sin.data_ptr(),
                _lib.ptr(positions), positions is not None and positions.dtype == torch.int64, cos.shape[0], S, B, n1, n2,
                D, 2 * cos.shape[1], not interleaved, eps, NATIVE_TYPES[qkv.dtype], _lib.stream_ptr())
        _lib.check(rc, "gfs_qk_norm_rope_bwd")
        if q_weight is not None:
            _lib.add_launches(1)      # the weights' gradients are added up in a launch of their own
        return dqkv, dw1, dw2, None, None, None, None, None, None, None


def qk_norm_rope(qkv: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, cos: torch.Tensor,
                 sin: torch.Tensor, num_heads: int, num_kv_heads: int, eps: float = 1e-5,
                 positions: torch.Tensor | None = None, interleaved: bool = True):
    """``qkv [S, B, (num_heads + 2 num_kv_heads) * D]`` -> ``(q [S, B, num_heads, D], k [S, B, num_kv_heads, D], v)``.

    q and k are normalised per head with ``q_weight``, ``k_weight [D]`` (of qkv's type; both ``None``: rotated only) and
    rotated as by :func:`~gpt_from_scratch_b200.ops.rope.rotary`, which documents ``cos``, ``sin``, ``positions`` and
    ``interleaved``; v is a view into ``qkv`` (not to be written to). Gradients for qkv and both weights. On CUDA:
    bfloat16, float16 or float32 and D up to 256, no forward-mode derivatives.
    """
    if num_heads < 0 or num_kv_heads < 0 or num_heads + num_kv_heads == 0:
        raise ValueError(f"qk_norm_rope: {num_heads} and {num_kv_heads} heads do not do")
    heads = num_heads + 2 * num_kv_heads
    if qkv.dim() != 3 or qkv.shape[2] == 0 or qkv.shape[2] % heads:
        raise ValueError(f"qk_norm_rope: qkv of shape {tuple(qkv.shape)} is not [S, B, {heads} * D]")
    S, B, W = qkv.shape
    D = W // heads
    check_tables("qk_norm_rope", qkv, cos, sin, positions, S, B, D)
    if not eps >= 0.0:
        raise ValueError(f"qk_norm_rope: eps {eps} is negative")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("qk_norm_rope: q and k are normalised both or not at all")
    for w in (q_weight, k_weight):
        if w is not None and (w.shape != (D,) or w.dtype != qkv.dtype or w.device != qkv.device):
            raise ValueError(f"qk_norm_rope: weights have to be {qkv.dtype} of shape [{D}] on {qkv.device}")
    if qkv.is_cuda:
        if q_weight is not None:
            q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
        args = (rows_of(qkv), q_weight, k_weight, cos.contiguous(), sin.contiguous(), num_heads, num_kv_heads, float(eps),
                None if positions is None else positions.contiguous(), bool(interleaved))
        return _forward(*args) if _lib.bare(qkv, q_weight, k_weight) else _QkNormRope.apply(*args)
    return qk_norm_rope_reference(qkv, q_weight, k_weight, cos, sin, num_heads, num_kv_heads, eps, positions, interleaved)
