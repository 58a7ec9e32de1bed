"""Blocks of a masked model that are called by themselves, without the model's mask, on the CPU."""
import pytest
import torch

from gpt_from_scratch_b200.config import GPTConfig
from gpt_from_scratch_b200.models.transformer_layer import TransformerLayer
from gpt_from_scratch_b200.ops import attention_mask
from gpt_from_scratch_b200.parallel import parallel_state as ps

CFG = dict(vocab_size=64, hidden_size=64, num_layers=1, num_attention_heads=4, max_position_embeddings=32, intermediate_size=128,
           init_method="normal", init_std=0.3)


@pytest.fixture(autouse=True)
def one_rank():
    ps.set_device("cpu")
    ps.initialize_parallel_state(1)
    ps.set_seed(3)


@pytest.mark.parametrize("more", [dict(qk_norm=True), dict(attention_softcap=0.5), dict(attention_window=3),
                                  dict(qk_norm=True, attention_softcap=5.0, attention_window=5)])
@pytest.mark.parametrize("dropout", [0.0, 0.3])
def test_a_block_by_itself_is_what_its_configuration_says(more, dropout):
    layer = TransformerLayer(0, GPTConfig(**CFG, **more, dropout_prob=dropout))
    if dropout:
        layer.eval()
    h = torch.randn(11, 2, 64, generator=torch.Generator().manual_seed(1))
    mask = attention_mask(2, 11, window=more.get("attention_window"))
    own, given = layer(h), layer(h, mask)
    assert torch.equal(own, given) and torch.equal(layer.attention(h), layer.attention(h, mask=mask))
    plain = TransformerLayer(0, GPTConfig(**CFG, dropout_prob=dropout))
    plain.load_state_dict(layer.state_dict(), strict=False)
    plain.eval()
    assert (plain(h) - own).abs().max() > 1e-3
    if more.get("qk_norm"):
        own.sum().backward()
        assert layer.attention.q_norm.weight.grad.abs().max() > 0


def test_a_block_cannot_know_documents():
    layer = TransformerLayer(0, GPTConfig(**CFG, eod_token_id=0, qk_norm=True))
    h = torch.randn(11, 2, 64, generator=torch.Generator().manual_seed(1))
    for call in (layer, layer.attention):
        with pytest.raises(ValueError, match="mask"):
            call(h)
    layer(h, attention_mask(2, 11, document_ids=torch.arange(22).view(2, 11) // 4))
