"""Model configuration. Field names and defaults follow the reference's ``GPTConfig``
(train.py:15-26); the extra fields select implementation details that the reference
hard-codes."""
from __future__ import annotations

from dataclasses import dataclass

from .ops.rope import RopeScaling


@dataclass
class GPTConfig:
    vocab_size: int = 50304          # GPT-2's 50257 padded so every TP size divides it
    hidden_size: int = 768
    num_layers: int = 12
    num_attention_heads: int = 12
    max_position_embeddings: int = 1024
    intermediate_size: int = 3072
    rms_norm_eps: float = 1e-5
    bias: bool = False
    dropout_prob: float = 0.0
    # --- additions ---
    rope_base: float = 10000.0
    init_method: str = "xavier_uniform"   # or "normal"
    init_std: float = 0.02
    attention_impl: str = "fused"         # "fused": tcgen05 flash attention on CUDA; "torch": eager oracle
    reference_quirks: bool = False        # reproduce reference behaviours that were fixed by default
    rope_scaling: RopeScaling | None = None  # angles for contexts longer than trained on (ops/rope.py)
    # Any of these four sends attention through ops/qk_norm_rope.py and ops/masked_attention.py (on CUDA their kernels in bf16 with
    # heads of 64 or 128, else their torch forms, as without the four; attention then makes its S x S matrix):
    qk_norm: bool = False                 # RMSNorm of every head of q and k, before the rotation
    attention_softcap: float = 0.0        # c > 0: scores become c tanh(score / c)
    attention_window: int = 0             # w > 0: no token sees one more than w - 1 before it
    eod_token_id: int = -1                # >= 0: documents end with it, tokens see (and count positions in) their own only

    def keys_per_token(self, seq_len: int) -> float:
        """Keys that a token of a whole sequence sees on average, the causal half of it (itself counted at half) or what the window
        leaves of that. Documents see less, by their lengths."""
        w = min(self.attention_window or seq_len, seq_len)
        return w - w * w / (2.0 * seq_len) if seq_len else 0.0

    def flops_per_token(self, seq_len: int, keys: float | None = None) -> float:
        """Forward+backward matmul FLOPs per token, of attention those for the ``keys`` that a token sees on average
        (:meth:`keys_per_token`)."""
        H, I, L, V = self.hidden_size, self.intermediate_size, self.num_layers, self.vocab_size
        keys = self.keys_per_token(seq_len) if keys is None else keys
        return 3.0 * (L * (2.0 * (4 * H * H + 3 * H * I) + 4.0 * keys * H) + 2.0 * H * V)

    def num_parameters(self) -> int:
        H, I, L, V = self.hidden_size, self.intermediate_size, self.num_layers, self.vocab_size
        qk = 2 * (H // self.num_attention_heads) if self.qk_norm else 0
        return 2 * V * H + L * (4 * H * H + 3 * H * I + 2 * H + qk) + H
