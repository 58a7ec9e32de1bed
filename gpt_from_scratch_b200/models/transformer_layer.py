"""Pre-norm transformer block with tensor-parallel attention and SwiGLU MLP.

Structure and parameter names follow the reference (core/transformer_layer.py:14-105):
``x + drop(attn(norm1(x)))`` then ``x + drop(mlp(norm2(x)))`` on ``[S/P, B, H]``
activations. The attention path keeps the projection output packed as
``[S, B, 3, nh/P, D]`` and hands it to the fused RoPE + flash-attention operator, so none
of the reference's permute/contiguous copies exist; with dropout disabled (the only value
the reference's CLI can reach) the residual adds run inside the row-parallel GEMMs.

With norms of q and k, capped scores, a window or documents (``config.qk_norm`` and the fields next to it) the packed
projection goes through :func:`~gpt_from_scratch_b200.ops.qk_norm_rope.qk_norm_rope` and
:func:`~gpt_from_scratch_b200.ops.masked_attention.masked_attention` instead, under a mask that the model makes once for
all blocks; a block that is called without one makes its own, except for documents, which it cannot know.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from ..ops.attention import attention_reference, fused_rope_attention
from ..ops.dropout import dropout_add
from ..ops.masked_attention import AttentionMask, attention_mask, masked_attention, masked_attention_reference
from ..ops.qk_norm_rope import qk_norm_rope, qk_norm_rope_reference
from ..ops.rope import rope_reference
from ..parallel import parallel_state as ps
from ..parallel.layers import ColumnParallelLinear, RowParallelLinear
from .init import get_init_method
from .mlp import ParallelMLP
from .normalization import RMSNorm
from .position_embeddings import RotaryEmbedding


def needs_mask(config) -> bool:
    """The configuration asks for what only masked attention computes."""
    return bool(getattr(config, "qk_norm", False) or getattr(config, "attention_softcap", 0.0) or
                getattr(config, "attention_window", 0) or getattr(config, "eod_token_id", -1) >= 0)


class ParallelAttention(nn.Module):
    def __init__(self, config):
        super().__init__()
        self.hidden_size = config.hidden_size
        self.num_attention_heads = config.num_attention_heads
        self.head_dim = self.hidden_size // self.num_attention_heads
        world = ps.get_tensor_model_parallel_world_size()
        assert self.num_attention_heads % world == 0, "heads must be divisible by the TP size"
        self.num_heads_per_partition = self.num_attention_heads // world
        bias = getattr(config, "bias", False)
        init_method = get_init_method(config)
        self.qkv_proj = ColumnParallelLinear(self.hidden_size, 3 * self.hidden_size, bias=bias,
                                             init_method=init_method)
        self.out_proj = RowParallelLinear(self.hidden_size, self.hidden_size, bias=bias, init_method=init_method)
        self.rotary_emb = RotaryEmbedding(self.head_dim, config.max_position_embeddings,
                                          getattr(config, "rope_base", 10000.0),
                                          round_to_activation_dtype=getattr(config, "reference_quirks", False),
                                          scaling=getattr(config, "rope_scaling", None))
        self.attention_impl = getattr(config, "attention_impl", "fused")
        self.softcap = getattr(config, "attention_softcap", 0.0)
        self.masked = needs_mask(config)
        self.window = getattr(config, "attention_window", 0)
        self.documents = getattr(config, "eod_token_id", -1) >= 0
        if getattr(config, "qk_norm", False):
            self.q_norm = RMSNorm(self.head_dim, config.rms_norm_eps)
            self.k_norm = RMSNorm(self.head_dim, config.rms_norm_eps)
        else:
            self.q_norm = self.k_norm = None

    def _masked(self, hidden_states, residual, mask: AttentionMask | None):
        nh, D = self.num_heads_per_partition, self.head_dim
        if mask is None and self.documents:
            raise ValueError("attention over documents (eod_token_id) needs the mask that the model makes of its tokens")
        qkv = self.qkv_proj(hidden_states)                 # [S, B, 3H/P]
        S, B, _ = qkv.shape
        if mask is None:
            mask = attention_mask(B, S, window=self.window or None, device=qkv.device)
        cos, sin = self.rotary_emb(qkv, S)
        if cos.dtype in (torch.bfloat16, torch.float16):   # a model that was cast as a whole
            cos, sin = cos.float(), sin.float()
        native = self.attention_impl == "fused" and (not qkv.is_cuda or
                                                     (qkv.dtype == torch.bfloat16 and D in (64, 128)))
        norm, attend = ((qk_norm_rope, masked_attention) if native else
                        (qk_norm_rope_reference, masked_attention_reference))
        normed = self.q_norm is not None
        q, k, v = norm(qkv, self.q_norm.weight if normed else None, self.k_norm.weight if normed else None, cos, sin, nh, nh,
                       eps=self.q_norm.eps if normed else 1e-5, positions=mask.positions)
        ctx = attend(q.permute(1, 2, 0, 3), k.permute(1, 2, 0, 3), v.permute(1, 2, 0, 3), mask, softcap=self.softcap)
        return self.out_proj(ctx.permute(2, 0, 1, 3).reshape(S, B, nh * D), residual)

    def forward(self, hidden_states, residual=None, mask: AttentionMask | None = None):
        if mask is not None or self.masked:
            return self._masked(hidden_states, residual, mask)
        nh, D = self.num_heads_per_partition, self.head_dim
        world = ps.get_tensor_model_parallel_world_size()
        S_full, B_ = hidden_states.shape[0] * world, hidden_states.shape[1]
        w = self.qkv_proj.weight
        rope_in_gemm = (self.attention_impl == "fused" and w.is_cuda and w.dtype == hidden_states.dtype ==
                        torch.bfloat16 and D in (64, 128) and self.qkv_proj.bias is None)
        if rope_in_gemm:
            # q and k are rotated by the projection GEMM's epilogue
            cos, sin = self.rotary_emb(hidden_states, S_full)
            qkv = self.qkv_proj(hidden_states, rope=(cos, sin, 2 * nh * D, D, B_))
        else:
            qkv = self.qkv_proj(hidden_states)             # [S, B, 3H/P]
        S, B, W = qkv.shape
        if not rope_in_gemm:
            cos, sin = self.rotary_emb(qkv, S)
        if self.attention_impl == "fused":
            ctx = fused_rope_attention(qkv.reshape(S * B, W), cos, sin, S, B, nh, D,
                                       pre_rotated=rope_in_gemm).view(S, B, nh * D)
        else:
            q, k, v = qkv.view(S, B, 3, nh, D).unbind(2)
            q, k = rope_reference(q, cos, sin), rope_reference(k, cos, sin)
            o = attention_reference(q.permute(1, 2, 0, 3), k.permute(1, 2, 0, 3), v.permute(1, 2, 0, 3), True)
            ctx = o.permute(2, 0, 1, 3).reshape(S, B, nh * D)
        return self.out_proj(ctx, residual)                # [S/P, B, H]


class TransformerLayer(nn.Module):
    def __init__(self, layer_id, config):
        super().__init__()
        self.layer_id = layer_id
        self.input_norm = RMSNorm(config.hidden_size, config.rms_norm_eps)
        self.attention = ParallelAttention(config)
        self.post_attention_norm = RMSNorm(config.hidden_size, config.rms_norm_eps)
        self.mlp = ParallelMLP(config)
        self.dropout_prob = getattr(config, "dropout_prob", 0.0)
        self.dropout = nn.Dropout(self.dropout_prob)

    def forward(self, hidden_states, mask: AttentionMask | None = None):
        if self.dropout_prob == 0.0 or not self.training:
            h, res = self.input_norm(hidden_states, fork=True)
            x = self.attention(h, residual=res, mask=mask) if mask is not None else self.attention(h, residual=res)
            h, res = self.post_attention_norm(x, fork=True)
            return self.mlp(h, residual=res)
        # residual + dropout(x) in one kernel (regenerated mask in the backward)
        h = self.input_norm(hidden_states)
        h = self.attention(h, mask=mask) if mask is not None else self.attention(h)
        x = dropout_add(h, hidden_states, self.dropout_prob, True)
        return dropout_add(self.mlp(self.post_attention_norm(x)), x, self.dropout_prob, True)
