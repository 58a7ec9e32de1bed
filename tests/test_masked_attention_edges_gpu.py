"""Masked attention at the edges of its arguments, against 64 bits. Tolerances: those of test_masked_attention_gpu.py, relative to values,
whatever their size."""
import math

import pytest
import torch
from test_masked_attention_gpu import bounds_and_values, check, run

from gpt_from_scratch_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,size", [(64, 5.0), (128, 3.5)])
@pytest.mark.parametrize("signs", ["cap", "negative cap", "both"])
@pytest.mark.parametrize("cap,exponent", [(50.0, 29), (50.0, -40), (55.0, 40), (55.0, -40), (900.0, 40), (900.0, -40)])
def test_saturated_scores_and_values_far_from_one(cuda_device, cap, exponent, signs, D, size):
    """Every score at +-200, which caps up to 55 bring to +-0.999 of themselves: probabilities are at their bounds before they are
    divided by their sum. Values of one to two times 2^exponent, within the range that the operator documents, of one sign, so that
    their sums grow with the keys. Its derivatives of capped scores
    are exact to a few 2^-24 of 4, and here they are above 2^-10 (or, for the large cap, near 1): 2^-12, the slack of the bounds."""
    B, nh, S = 1, 2, 2000
    gen = torch.Generator(device="cuda").manual_seed(D)

    def sign(*shape):
        return torch.randint(0, 2, shape, device="cuda", generator=gen) * 2.0 - 1.0
    direction = sign(D) * 5.0
    turn = {"cap": torch.ones(S, 1, device="cuda"), "negative cap": -torch.ones(S, 1, device="cuda"), "both": sign(S, 1)}[signs]
    q = direction.expand(B, nh, S, D).bfloat16()
    k = (direction / 5.0 * size * turn).expand(B, nh, S, D).bfloat16()
    v = ((1 + torch.rand(B, nh, S, D, device="cuda", generator=gen)) * 2.0 ** exponent).bfloat16()
    dout = torch.randn(B, nh, S, D, device="cuda", generator=gen).bfloat16()
    mask = ops.attention_mask(B, S, device="cuda")
    want, tols = bounds_and_values(q, k, v, dout, mask.visible(), cap, None, 1 / math.sqrt(D))
    check(run(q, k, v, dout, mask, softcap=cap), want, tols, f"cap {cap} {signs}")
