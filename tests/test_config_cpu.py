"""The configuration's interface and its count of operations, on the CPU."""
import json

import numpy as np
import pytest

from gpt_from_scratch_b200.config import GPTConfig


def test_positional_arguments_keep_their_places():
    """The order that the fields had before those of the masked path, which stand behind them."""
    cfg = GPTConfig(512, 64, 2, 4, 32, 128, 1e-6, True, 0.1, 5000.0, "normal", 0.1, "torch", True)
    assert cfg == GPTConfig(vocab_size=512, hidden_size=64, num_layers=2, num_attention_heads=4, max_position_embeddings=32,
                            intermediate_size=128, rms_norm_eps=1e-6, bias=True, dropout_prob=0.1, rope_base=5000.0,
                            init_method="normal", init_std=0.1, attention_impl="torch", reference_quirks=True)
    assert cfg.rope_scaling is None and not cfg.qk_norm


@pytest.mark.parametrize("S,window", [(1, 0), (100, 0), (100, 1), (100, 30), (100, 100), (100, 250)])
def test_operations_count_the_keys_that_are_seen(S, window):
    cfg = GPTConfig(hidden_size=64, num_layers=3, attention_window=window)
    keys = sum(min(i + 1, window or S) for i in range(S)) / S
    # the token itself counts at half, so a half may be missing
    assert 0 <= keys - cfg.keys_per_token(S) <= 0.5
    attention = cfg.flops_per_token(S) - cfg.flops_per_token(S, 0.0)
    assert attention == pytest.approx(3 * 3 * 4 * 64 * cfg.keys_per_token(S))
    if not window:
        assert cfg.keys_per_token(S) == S / 2


@pytest.mark.parametrize("window", [0, 4])
def test_logged_utilisation_counts_documents(tmp_path, window):
    """One step on tokens that are known; the log's utilisation over its tokens a second is the count of operations."""
    import train
    tokens = np.full(2 * 16 + 1, 3, dtype=np.uint16)
    tokens[[4, 5, 15, 27]] = 0          # sequences of documents of 5, 1, 10 and of 12, 4 tokens
    tokens.tofile(tmp_path / "tokens.bin")
    argv = ["--vocab-size", "64", "--hidden-size", "32", "--num-layers", "1", "--num-attention-heads", "4",
            "--intermediate-size", "48", "--seq-len", "16", "--max-position-embeddings", "16", "--batch-size", "2",
            "--num-workers", "0", "--device", "cpu", "--log-interval", "1", "--max-steps", "1", "--eod-token-id", "0",
            "--attention-window", str(window), "--peak-tflops", "0.5", "--heartbeat-timeout", "0", "--data-path",
            str(tmp_path / "tokens.bin"), "--log-jsonl", str(tmp_path / "log.jsonl")]
    train.main(argv)
    rec = json.loads((tmp_path / "log.jsonl").read_text().splitlines()[0])
    cfg = train.build_config(train.parse_args(argv))
    pairs = sum(min(i + 0.5, window or 16) for n in (5, 1, 10, 12, 4) for i in range(n))
    assert rec["mfu"] * 0.5e12 / rec["tokens_per_sec"] == pytest.approx(cfg.flops_per_token(16, pairs / 32), rel=1e-5)
    assert cfg.flops_per_token(16, pairs / 32) < cfg.flops_per_token(16)
