"""Sizes and scales that the kernels' 32 bits cannot hold are refused before a kernel is asked, on the CPU too."""
import pytest
import torch

from gpt_from_scratch_b200 import ops


@pytest.mark.parametrize("batch,seq_len", [(2 ** 32 + 1, 1), (2 ** 31, 1), (1, 2 ** 30), (1, 2 ** 32 + 5), (-1, 4), (4, -1)])
def test_masks_past_32_bits(batch, seq_len):
    with pytest.raises(ValueError):
        ops.attention_mask(batch, seq_len, device="meta")


@pytest.mark.parametrize("batch,seq_len", [(1.0, 4), (2, 4.0)])
def test_sizes_are_whole_numbers(batch, seq_len):
    with pytest.raises(TypeError):
        ops.attention_mask(batch, seq_len)


@pytest.mark.parametrize("scale", [1e300, 1e31, 1e-31, 5e-324, 0.0, -1.0, float("inf"), float("nan")])
@pytest.mark.parametrize("softcap", [0.0, 1e-6])
def test_scales_past_32_bits(scale, softcap):
    x = torch.randn(1, 2, 5, 8)
    mask = ops.attention_mask(1, 5)
    with pytest.raises(ValueError):
        ops.masked_attention(x, x, x, mask, scale=scale, softcap=softcap)
    for fits in (1e-30, 1e30):
        ops.masked_attention(x, x, x, mask, scale=fits, softcap=softcap)
