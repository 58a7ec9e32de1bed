"""Masked attention at the edges of its arguments, against 64 bits. Tolerances: those of test_masked_attention_gpu.py, relative to values,
whatever their size."""
import math

import pytest
import torch
from test_masked_attention_gpu import bounds_and_values, check, document_ids, run, tensors

from gpt_from_scratch_b200 import ops
from gpt_from_scratch_b200.ops.masked_attention import _layout

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


@pytest.mark.parametrize("S", [1, 63, 128, 129, 130, 257, 385, 640, 1025, 3001])
@pytest.mark.parametrize("kind", ["none", "docs", "padded", "empty", "end"])
@pytest.mark.parametrize("causal,window", [(True, None), (True, 7), (True, 200), (False, None)])
def test_pairs_of_tiles(cuda_device, S, kind, causal, window):
    """Every pair of query tiles once; the blocks of 64 keys of each tile hold what its rows see, none of them is empty, and the blocks of
    both are one stretch. end: the last token alone is padding."""
    B = 2
    if kind == "end":
        ids = torch.zeros(B, S, dtype=torch.int64, device=cuda_device)
        ids[:, -1] = -1
    else:
        ids = document_ids(B, S, kind, S)
    mask = ops.attention_mask(B, S, causal, ids, None, window, device=cuda_device)
    n, at = ((S + 127) // 128 + 1) // 2, _layout(B, S)["pairs"]
    pairs = mask.buffer[at:at + B * n * 8].view(B, n, 8).cpu()
    first, last = mask.first.cpu(), mask.last.cpu()
    for b in range(B):
        assert sorted(pairs[b, :, 0].tolist()) == list(range(n))
        for t, a0, a1, b0, b1, padded, _, _ in pairs[b].tolist():
            assert bool(padded) == (ids is not None and bool((ids[b] < 0).any()))
            tiles = [(t * 256, a0, a1)]
            if t * 256 + 128 < S:
                tiles.append((t * 256 + 128, b0, b1))
                assert max(a0, b0) <= min(a1, b1)              # no gap
            else:
                assert b0 == b1
            for row, j0, j1 in tiles:
                assert 0 <= j0 < j1 <= (S + 63) // 64
                rows = slice(row, min(row + 128, S))
                seen = first[b, rows] < last[b, rows]
                assert (first[b, rows][seen] >= j0 * 64).all() and (last[b, rows][seen] <= j1 * 64).all()


@pytest.mark.parametrize("S", [129, 257, 385])
@pytest.mark.parametrize("nh,nkv,D", [(2, 2, 64), (3, 1, 128), (4, 2, 64)])
def test_a_last_tile_of_one_padding_token(cuda_device, S, nh, nkv, D):
    ids = torch.zeros(2, S, dtype=torch.int64, device=cuda_device)
    ids[:, -1] = -1
    ids[1, S // 2:] = -1
    mask = ops.attention_mask(2, S, document_ids=ids)
    q, k, v, dout = tensors(2, nh, nkv, S, D, S, packed=False)
    want, tols = bounds_and_values(q, k, v, dout, mask.visible(), 0.0, None, 1 / math.sqrt(D))
    got = run(q, k, v, dout, mask)
    check(got, want, tols)
    hidden = (ids < 0)[:, None, :, None]
    assert all((t.masked_select(hidden) == 0).all() for t in got)
