"""The configuration's interface and its count of operations, on the CPU."""
from gpt_from_scratch_b200.config import GPTConfig


def test_positional_arguments_keep_their_places():
    """The order that the fields had before those of the masked path, which stand behind them."""
    cfg = GPTConfig(512, 64, 2, 4, 32, 128, 1e-6, True, 0.1, 5000.0, "normal", 0.1, "torch", True)
    assert cfg == GPTConfig(vocab_size=512, hidden_size=64, num_layers=2, num_attention_heads=4, max_position_embeddings=32,
                            intermediate_size=128, rms_norm_eps=1e-6, bias=True, dropout_prob=0.1, rope_base=5000.0,
                            init_method="normal", init_std=0.1, attention_impl="torch", reference_quirks=True)
    assert cfg.rope_scaling is None and not cfg.qk_norm
