"""Attention under a mask of documents, prefix, window and padding, with capped or distance-biased scores
(csrc/masked_attention.cu, csrc/masked_attention_bwd.cu), and its torch oracle.

The mask is made once per batch (:func:`attention_mask`) and used by every layer and by the backward pass: what a query
sees is one range of keys, whose ends grow along the sequence, so the mask is two numbers per token, and the kernels skip every
block that it hides.
"""
from __future__ import annotations

import ctypes
import functools
import math
import operator

import torch

from . import _lib


class AttentionMask:
    """What :func:`attention_mask` returns. ``first``, ``last``: int32 ``[B, S]``, query s sees the keys ``[first, last)`` (none:
    padding); ``positions``: int32 ``[B, S]``, the place of every token in its document (for
    :func:`~gpt_from_scratch_b200.ops.rope.rotary`)."""
    __slots__ = ("batch", "seq_len", "device", "buffer", "_parts")

    def __init__(self, batch: int, seq_len: int, device: torch.device, buffer: torch.Tensor | None = None, parts=None):
        self.batch, self.seq_len, self.device = batch, seq_len, device
        self.buffer = buffer        # CUDA: what the kernels read (gfs_attention_mask); its parts are cut out when asked for
        self._parts = parts

    def _part(self, i: int) -> torch.Tensor:
        if self._parts is not None:
            return self._parts[i]
        B, S = self.batch, self.seq_len
        layout = _layout(B, S)
        if i == 2:
            return self.buffer.as_strided((B, S), (S, 1), layout["positions"])
        return self.buffer.as_strided((B, S), (_pad128(S), 1), layout["last" if i else "first"])

    @property
    def first(self) -> torch.Tensor:
        return self._part(0)

    @property
    def last(self) -> torch.Tensor:
        return self._part(1)

    @property
    def positions(self) -> torch.Tensor:
        return self._part(2)

    def visible(self) -> torch.Tensor:
        """bool ``[B, S, S]``, query by key."""
        at = torch.arange(self.seq_len, device=self.device)
        return (at >= self.first.unsqueeze(-1)) & (at < self.last.unsqueeze(-1))


@functools.lru_cache(maxsize=256)
def _layout(B: int, S: int) -> dict[str, int]:
    """Where a mask's buffer has its parts, and its length."""
    at = (ctypes.c_longlong * 10)()
    _lib.lib().gfs_attention_mask_layout(B, S, at)
    return dict(zip(("first", "last", "qfirst", "qlast", "plan_q", "plan_k", "pairs", "padded", "positions", "end"), at))


def _pad128(S: int) -> int:
    return (S + 127) // 128 * 128


def _mask_reference(batch, seq_len, causal, ids, prefix, window, device):
    S = seq_len
    at = torch.arange(S, device=device).expand(batch, S)
    edge = at == 0
    if ids is not None:
        edge = edge | (ids != ids.roll(1, dims=1))

    def following(stop):      # the first stop behind every token, S where there is none
        after = torch.cat((torch.where(stop, at, S)[:, 1:], torch.full((batch, 1), S, device=device)), dim=1)
        return after.flip(1).cummin(dim=1).values.flip(1) if S else after[:, :0]
    start = torch.where(edge, at, 0).cummax(dim=1).values if S else at
    first, last = start, at + 1 if causal else following(edge)
    if prefix is not None:
        plain = torch.where(prefix, -1, at).cummax(dim=1).values if S else at
        lead = prefix & (plain < start)
        last = torch.where(lead, following(edge | ~prefix), last)
    if window is not None:
        first = torch.maximum(first, at - window + 1)
    if ids is not None:
        first, last = torch.where(ids < 0, at, first), torch.where(ids < 0, at, last)
    return AttentionMask(batch, S, device, parts=(first.int(), last.int(), (at - start).int()))


def _mask_buffer(B, S, ids, prefix, causal, window, device) -> torch.Tensor:
    buffer = torch.empty(_layout(B, S)["end"], dtype=torch.int32, device=device)
    with _lib.on_device(buffer), _lib.nvtx("attention_mask"):
        rc = _lib.lib().gfs_attention_mask(_lib.ptr(ids), ids is not None and ids.dtype == torch.int64, _lib.ptr(prefix), B,
                                           S, causal, window, buffer.data_ptr(), _lib.stream_ptr())
    _lib.check(rc, "gfs_attention_mask")
    return buffer


class _MaskBuffer(torch.autograd.Function):
    """For traces, which see a function where they miss a pointer."""
    @staticmethod
    def forward(ctx, *args):
        buffer = _mask_buffer(*args)
        ctx.mark_non_differentiable(buffer)
        return buffer


def attention_mask(batch: int, seq_len: int, causal: bool = True, document_ids: torch.Tensor | None = None,
                   prefix_mask: torch.Tensor | None = None, window: int | None = None, device=None) -> AttentionMask:
    """The mask of ``batch`` sequences of ``seq_len`` tokens for :func:`masked_attention`.

    ``document_ids`` (int32 or int64 ``[B, S]``): tokens see only their own document, a run of equal numbers; a run of negative
    ones is padding, which sees nothing and is seen by nothing. ``causal``: a token sees those up to itself, else all of its
    document. ``prefix_mask`` (bool ``[B, S]``, causal only): the tokens at the head of a document that are marked are seen
    by all of it. ``window`` (causal only): a token sees no token more than ``window - 1`` before it. ``device`` defaults to
    the tensors' one, without tensors to the CPU. On CUDA one launch.
    """
    batch, seq_len = operator.index(batch), operator.index(seq_len)      # (in traces, sizes are tensors)
    if not (0 <= batch < 2 ** 31 and 0 <= seq_len <= 0x3fff0000):       # 32-bit places, also behind a window
        raise ValueError(f"attention_mask: {batch} sequences of {seq_len} tokens do not do")
    if document_ids is not None and (document_ids.shape != (batch, seq_len) or
                                     document_ids.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"attention_mask: document_ids have to be int32 or int64 of shape [{batch}, {seq_len}]")
    if prefix_mask is not None and (prefix_mask.shape != (batch, seq_len) or prefix_mask.dtype != torch.bool):
        raise ValueError(f"attention_mask: prefix_mask has to be bool of shape [{batch}, {seq_len}]")
    if window is not None and window < 1:
        raise ValueError(f"attention_mask: a window of {window} tokens leaves nothing to see")
    if not causal and (prefix_mask is not None or window is not None):
        raise ValueError("attention_mask: prefix_mask and window go with causal masks")
    given = [t.device for t in (document_ids, prefix_mask) if t is not None]
    device = torch.device(device) if device is not None else (given[0] if given else torch.device("cpu"))
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    if any(d != device for d in given):
        raise ValueError(f"attention_mask: document_ids and prefix_mask have to be on {device}")
    if device.type != "cuda":
        return _mask_reference(batch, seq_len, causal, document_ids, prefix_mask, window, device)
    ids = None if document_ids is None else document_ids.contiguous()
    prefix = None if prefix_mask is None else prefix_mask.contiguous()
    make = _mask_buffer if _lib.bare(ids, prefix) else _MaskBuffer.apply
    return AttentionMask(batch, seq_len, device, make(batch, seq_len, ids, prefix, causal, min(window or 0, 0x7fffffff), device))


def masked_attention_reference(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: AttentionMask, softcap: float = 0.0,
                               alibi_slopes: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """:func:`masked_attention` in torch operations (materialises the S x S matrix): fp32, 64 bits for 64-bit inputs."""
    nh, nkv, S, D = q.shape[1], k.shape[1], q.shape[2], q.shape[3]
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    k, v = (t.to(wide).repeat_interleave(nh // nkv, dim=1) for t in (k, v))
    s = torch.matmul(q.to(wide), k.transpose(-1, -2)) * (1.0 / math.sqrt(D) if scale is None else scale)
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if alibi_slopes is not None:
        at = torch.arange(S, device=q.device)
        s = s - alibi_slopes.to(wide)[:, None, None] * (at[:, None] - at).abs()
    see = mask.visible().unsqueeze(1)
    empty = ~see.any(-1, keepdim=True)
    p = torch.softmax(s.masked_fill(~see & ~empty, float("-inf")), dim=-1).masked_fill(empty, 0.0)
    return torch.matmul(p, v).to(q.dtype)


@functools.lru_cache(maxsize=1024)
def _strides(shape, stride) -> tuple[int, int, int]:
    """Element strides (sequence, batch, head) of a ``[B, heads, S, D]`` tensor; those of single entries, which lead
    nowhere, are given as the kernels want them."""
    (nb, nh, ns, d), (b, h, s, _) = shape, stride
    return s if ns > 1 else d, b if nb > 1 else d, h if nh > 1 else d


@functools.lru_cache(maxsize=1024)
def _stride_array(*layouts):
    """ctypes array of the strides of tensors given as shape, stride, shape, stride, ..."""
    flat = [n for shape, stride in zip(layouts[::2], layouts[1::2]) for n in _strides(shape, stride)]
    return (ctypes.c_longlong * len(flat))(*flat)


@functools.lru_cache(maxsize=1024)
def _steps_of_16_bytes(shape, stride) -> bool:
    return stride[3] == 1 and all(s > 0 and s % 8 == 0 for s in _strides(shape, stride))


def _readable(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself if the kernels can read its layout (16-byte steps, no broadcast dimensions), else a contiguous copy."""
    if not t.data_ptr() % 16 and _steps_of_16_bytes(t.shape, t.stride()):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _forward(q, k, v, buffer, slopes, softcap: float, scale: float, training: bool):
    B, nh, S, D = q.shape
    out = torch.empty_like(q)
    # for the backward: 32 bits per row (the log of its sum) and 8 bits per number (what rounding leaves out of ``out``)
    saved = torch.empty(B * nh * _pad128(S) * (1 + D // 4), dtype=torch.float32, device=q.device) if training else None
    kv = k.shape
    st = _stride_array(q.shape, q.stride(), kv, k.stride(), kv, v.stride(), q.shape, out.stride())
    with _lib.on_device(q), _lib.nvtx("masked_attention_fwd"):
        rc = _lib.lib().gfs_masked_attention_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _lib.ptr(saved),
                                                 buffer.data_ptr(), S, B, nh, kv[1], D, st, scale, softcap,
                                                 _lib.ptr(slopes), _lib.stream_ptr())
    _lib.check(rc, "gfs_masked_attention_fwd")
    return out, saved


@functools.lru_cache(maxsize=256)
def _scratch(S: int, B: int, nh: int, nkv: int, D: int, device: int = 0) -> int:
    """fp32 elements that the backward wants on ``device``, the current one (it depends on the number of its SMs)."""
    return _lib.lib().gfs_masked_attention_scratch(S, B, nh, nkv, D)


class _MaskedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, buffer, slopes, softcap, scale):
        q, k, v = _readable(q), _readable(k), _readable(v)
        out, saved = _forward(q, k, v, buffer, slopes, softcap, scale, True)
        ctx.save_for_backward(q, k, v, out, saved, buffer, slopes)
        ctx.args = (softcap, scale)
        ctx.traced = torch._C._is_tracing()
        return out

    @staticmethod
    @_lib.first_order
    def backward(ctx, dout):
        q, k, v, out, saved, buffer, slopes = ctx.saved_tensors
        softcap, scale = ctx.args
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        if q.numel() == 0:
            return dq, dk.zero_(), dv.zero_(), None, None, None, None
        B, nh, S, D = shape = q.shape
        kv = k.shape
        dout = _readable(dout)
        dvec = torch.empty(B * nh * _pad128(S), dtype=torch.float32, device=q.device)
        st = _stride_array(shape, q.stride(), kv, k.stride(), kv, v.stride(), shape, out.stride(), shape, dout.stride(), shape,
                           dq.stride(), kv, dk.stride(), kv, dv.stride())
        with _lib.on_device(q), _lib.nvtx("masked_attention_bwd"):
            scratch = _scratch(S, B, nh, kv[1], D, q.get_device())
            partial = torch.empty(scratch, dtype=torch.float32, device=q.device) if scratch else None
            rc = _lib.lib().gfs_masked_attention_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                                     dout.data_ptr(), saved.data_ptr(), dvec.data_ptr(), _lib.ptr(partial),
                                                     scratch, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), buffer.data_ptr(), S, B,
                                                     nh, kv[1], D, st, scale, softcap, _lib.ptr(slopes), _lib.stream_ptr())
        _lib.check(rc, "gfs_masked_attention_bwd")
        _lib.add_launches(3 if scratch else 2)  # pre-pass + two main kernels (+ the sum of the parts)
        return dq, dk, dv, None, None, None, None


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: AttentionMask, softcap: float = 0.0,
                     alibi_slopes: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """Attention of ``q [B, heads, S, D]`` over ``k``, ``v [B, kv_heads, S, D]`` under ``mask`` (:func:`attention_mask`).

    Heads of q share those of k and v in groups of ``heads / kv_heads``. Scores are ``scale * q k`` (default ``1 / sqrt(D)``), with
    ``softcap`` c > 0 ``c tanh(scale * q k / c)``, with ``alibi_slopes`` (fp32 ``[heads]``, constants for autograd) minus
    ``slope * |i - j|``. A query that sees nothing gets zeros, and what padding holds does not matter. The result is laid out
    like q. On CUDA: bfloat16, D 64 or 128 and softcap up to 1000, any strides (copied first where a dimension is broadcast or
    16-byte accesses do not reach), deterministic, no forward-mode derivatives; other devices: torch operations.

    On CUDA probabilities and the gradients of scores are rounded to bfloat16 before their products. With a softcap of up to 50
    magnitudes of v, where not 0, have to lie between 2^-40, below which digits are lost where all of a query's scores are near the
    negative cap, and 2^30, above which sums may overflow where they are near the cap. A value that is not finite, outside of padding,
    may spread past the mask: a key's to all queries of a tile of 128 of which one sees any of the 64 keys of its block, and a
    query's to the gradients of such keys.
    """
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f"masked_attention: shapes {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)} do not fit")
    B, nh, S, D = q.shape
    nkv = k.shape[1]
    if (k.shape[0], k.shape[2], k.shape[3]) != (B, S, D) or nkv == 0 or nh % nkv:
        raise ValueError(f"masked_attention: k and v of shape {tuple(k.shape)} do not fit q of shape {tuple(q.shape)}")
    if (mask.batch, mask.seq_len) != (B, S):
        raise ValueError(f"masked_attention: a mask of {mask.batch} x {mask.seq_len} tokens for {B} x {S}")
    if not (q.dtype == k.dtype == v.dtype) or not (q.device == k.device == v.device == mask.device):
        raise ValueError("masked_attention: q, k and v have to be of one type and, with the mask, on one device")
    if not (softcap >= 0.0 and math.isfinite(softcap)):
        raise ValueError(f"masked_attention: softcap {softcap} is neither 0 nor positive")
    scale = 1.0 / math.sqrt(D) if scale is None and D else scale
    if scale is not None and not 1e-30 <= scale <= 1e30:
        raise ValueError(f"masked_attention: scale {scale} is not positive, or so far from 1 that 32 bits cannot hold it with a cap")
    if alibi_slopes is not None:
        if alibi_slopes.shape != (nh,) or alibi_slopes.dtype != torch.float32 or alibi_slopes.device != q.device:
            raise ValueError(f"masked_attention: alibi_slopes have to be fp32 of shape [{nh}] on {q.device}")
        if alibi_slopes.requires_grad:
            raise ValueError("masked_attention: alibi_slopes get no gradient")
    if q.is_cuda:
        if q.dtype != torch.bfloat16 or D not in (64, 128):
            raise ValueError(f"masked_attention: no native kernel for {q.dtype} and head_dim {D} (bfloat16 and 64 or 128 have "
                             "one); use masked_attention_reference for others")
        if softcap and not 1e-6 <= softcap <= 1e3:
            raise ValueError(f"masked_attention: softcap {softcap} is outside of 1e-6 to 1e3 (the error of a capped score is "
                             "2^-22 of the cap)")
        if B > 65535 or _pad128(S) * nh >= 2 ** 30 or _pad128(S) // 128 * B * nh >= 2 ** 31:
            raise ValueError(f"masked_attention: {B} sequences of {S} tokens with {nh} heads are too many for one call")
        slopes = None if alibi_slopes is None else alibi_slopes.contiguous()
        if _lib.bare(q, k, v):
            return _forward(_readable(q), _readable(k), _readable(v), mask.buffer, slopes, float(softcap), float(scale), False)[0]
        return _MaskedAttention.apply(q, k, v, mask.buffer, slopes, float(softcap), float(scale))
    return masked_attention_reference(q, k, v, mask, softcap, alibi_slopes, scale)
