"""The mask of masked attention, its refusals and its torch form, on the CPU; rotary positions and norms likewise."""
import math

import pytest
import torch

from gpt_from_scratch_b200 import ops


def by_hand(ids, prefix, causal, window):
    """[S, S] from the definition, token by token."""
    S = len(ids)
    see = torch.zeros(S, S, dtype=torch.bool)
    run = [0] * S
    for i in range(1, S):
        run[i] = run[i - 1] + (ids[i] != ids[i - 1])
    lead = [False] * S
    for i in range(S):
        lead[i] = prefix[i] and (i == 0 or run[i] != run[i - 1] or lead[i - 1])
    for i in range(S):
        for j in range(S):
            if run[i] != run[j] or ids[i] < 0:
                continue
            ok = not causal or j <= i or (lead[i] and lead[j]) or (lead[j] and not lead[i] and j <= i)
            if window is not None and j < i - window + 1:
                ok = False
            see[i, j] = ok
    return see


CASES = [
    ([0] * 9, [0] * 9, True, None),
    ([0] * 9, [0] * 9, False, None),
    ([5], [1], True, 1),
    ([3, 3, 3, 1, 1, 1, 1, 1, 9], [0] * 9, True, None),
    ([3, 3, 3, 1, 1, 1, 1, 1, 9], [1, 1, 0, 1, 1, 1, 0, 1, 1], True, None),
    ([3, 3, 3, 1, 1, 1, 1, 1, 9], [0, 1, 1, 1, 1, 1, 1, 1, 0], True, 3),
    ([3, 3, 3, 1, 1, 3, 3, -1, -1], [0] * 9, False, None),
    ([-1, 2, 2, -4, -4, 2, 2, 2, -1], [1] * 9, True, 2),
    ([-1] * 9, [0] * 9, True, None),
    ([0] * 9, [1] * 9, True, None),
    ([0] * 9, [0] * 9, True, 4),
]


@pytest.mark.parametrize("ids,prefix,causal,window", CASES)
def test_mask_follows_its_definition(ids, prefix, causal, window):
    p = torch.tensor([prefix], dtype=torch.bool)
    mask = ops.attention_mask(1, len(ids), causal, torch.tensor([ids]), p if causal else None, window)
    want = by_hand(ids, prefix if causal else [0] * len(ids), causal, window)
    assert torch.equal(mask.visible()[0], want)
    start = [max(j for j in range(i + 1) if j == 0 or ids[j] != ids[j - 1]) for i in range(len(ids))]
    assert mask.positions[0].tolist() == [i - s for i, s in enumerate(start)]
    assert (mask.first[0].diff() >= 0).all() and (mask.last[0].diff() >= 0).all()


def test_masked_attention_is_plain_attention_without_a_mask():
    q, k, v = (torch.randn(2, 3, 17, 8, dtype=torch.float64) for _ in range(3))
    for causal in (True, False):
        got = ops.masked_attention(q, k, v, ops.attention_mask(2, 17, causal))
        want = ops.attention_reference(q.float(), k.float(), v.float(), causal)
        assert (got.float() - want).abs().max() < 1e-5


def test_masked_attention_cpu_by_hand():
    """Shared heads, cap, distance and an empty row, one query at a time."""
    torch.manual_seed(0)
    q, k, v = torch.randn(1, 4, 7, 8).double(), torch.randn(1, 2, 7, 8).double(), torch.randn(1, 2, 7, 8).double()
    ids = torch.tensor([[1, 1, 1, 0, 0, -1, -1]])
    mask = ops.attention_mask(1, 7, True, ids)
    slopes = torch.tensor([0.5, 0.25, 0.125, 1.0])
    out = ops.masked_attention(q, k, v, mask, softcap=2.0, alibi_slopes=slopes)
    for h in range(4):
        for i in range(7):
            keys = [j for j in range(i + 1) if ids[0, j] == ids[0, i] >= 0]
            if not keys:
                assert (out[0, h, i] == 0).all()
                continue
            s = torch.tensor([2 * math.tanh(float(q[0, h, i] @ k[0, h // 2, j]) / math.sqrt(8) / 2) -
                              float(slopes[h]) * (i - j) for j in keys]).double()
            want = torch.softmax(s, 0) @ v[0, h // 2, keys]
            assert (out[0, h, i] - want).abs().max() < 1e-6


def test_refusals():
    ids = torch.zeros(2, 5, dtype=torch.int64)
    for args in (dict(document_ids=ids[:1]), dict(document_ids=ids.float()), dict(prefix_mask=ids),
                 dict(prefix_mask=torch.zeros(2, 4, dtype=torch.bool)), dict(window=0), dict(causal=False, window=3),
                 dict(causal=False, prefix_mask=ids.bool())):
        with pytest.raises(ValueError):
            ops.attention_mask(2, 5, **args)
    with pytest.raises(ValueError):
        ops.attention_mask(-1, 5)
    mask = ops.attention_mask(2, 5, document_ids=ids)
    q, k = torch.randn(2, 4, 5, 8), torch.randn(2, 2, 5, 8)
    ops.masked_attention(q, k, k, mask)
    bad = [(q[0], k, k, mask), (q, k, k[:, :1], mask), (q[:, :3], k, k, mask), (q, k[:, :, :4], k[:, :, :4], mask),
           (q, k.double(), k, mask), (q, k, k, ops.attention_mask(2, 6)), (q, k[..., :4], k[..., :4], mask)]
    for args in bad:
        with pytest.raises(ValueError):
            ops.masked_attention(*args)
    for kw in (dict(softcap=-1.0), dict(softcap=float("inf")), dict(softcap=float("nan")), dict(scale=0.0), dict(scale=-1.0),
               dict(alibi_slopes=torch.ones(2)), dict(alibi_slopes=torch.ones(4).double()),
               dict(alibi_slopes=torch.ones(4, requires_grad=True))):
        with pytest.raises(ValueError):
            ops.masked_attention(q, k, k, mask, **kw)


def test_rope_tables_and_refusals():
    cos, sin = ops.rope_tables(9, 8)
    want = torch.outer(torch.arange(9.0).double(), 10000.0 ** (-torch.arange(0, 8, 2).double() / 8))
    assert torch.equal(cos, want.cos().float()) and torch.equal(sin, want.sin().float())
    # a far position keeps its digits: the angle is formed in 64 bits
    cos, _ = ops.rope_tables(1_000_001, 2, base=10000.0)
    assert abs(float(cos[1_000_000, 0]) - math.cos(1_000_000.0)) < 2.0 ** -24
    # linear: position p of the long table is position p / factor of the short one
    long, short = ops.rope_tables(16, 8, scaling=ops.RopeScaling("linear", 4.0))[0], ops.rope_tables(4, 8)[0]
    assert (long[::4] - short).abs().max() < 2.0 ** -23
    # ntk: the fastest pair stays, the slowest is divided by the factor
    base = ops.rope_tables(3, 8)[1]
    ntk = ops.rope_tables(3, 8, scaling=ops.RopeScaling("ntk", 4.0))[1]
    assert torch.equal(ntk[:, 0], base[:, 0]) and abs(math.asin(float(ntk[1, 3])) * 4 - math.asin(float(base[1, 3]))) < 1e-9
    # by parts: a pair that turns more than `high` times in the original length stays, one below `low` is divided
    parts = ops.rope_tables(3, 8, scaling=ops.RopeScaling("by_parts", 4.0, original_length=100, low=1, high=8))[1]
    assert torch.equal(parts[:, 0], base[:, 0]) and abs(float(parts[1, 3]) * 4 - float(base[1, 3])) < 1e-7
    mid = ops.rope_tables(2, 8, scaling=ops.RopeScaling("by_parts", 4.0, original_length=100, low=1, high=8))[1][1, 1]
    turns = 100 * 0.1 / (2 * math.pi)
    keep = (turns - 1) / 7
    assert abs(float(mid) - math.sin(0.1 * keep + 0.1 / 4 * (1 - keep))) < 2.0 ** -23
    m = ops.rope_tables(2, 8, scaling=ops.RopeScaling("linear", 4.0, magnitude=None))[0][0, 0]
    assert abs(float(m) - (0.1 * math.log(4.0) + 1.0)) < 2.0 ** -23
    for bad in (dict(kind="other", factor=2.0), dict(kind="linear", factor=0.0), dict(kind="by_parts", factor=2.0)):
        with pytest.raises(ValueError):
            ops.RopeScaling(**bad)
    for bad in ((4, 7), (4, 0), (-1, 8)):
        with pytest.raises(ValueError):
            ops.rope_tables(*bad)


def test_rotary_refusals_and_reference():
    cos, sin = ops.rope_tables(6, 8)
    x = torch.randn(6, 2, 3, 8)
    assert (ops.rotary(x, cos, sin) - ops.apply_rope(x, cos, sin)).abs().max() < 1e-6
    half = ops.rotary(x, cos, sin, interleaved=False)
    order = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7])       # the same rotation with the pairs laid out apart
    assert (half[..., order] - ops.rotary(x[..., order], cos, sin)).abs().max() < 1e-6
    at = torch.zeros(2, 6, dtype=torch.int32)
    for args in ((x[0], cos, sin), (x[..., :4], cos, sin), (x, cos[:5], sin[:5]), (x, cos, sin[:, :2]), (x, cos.double(), sin.double()),
                 (x, cos, sin, at[:1]), (x, cos, sin, at.float()), (x, cos, sin, at - 1), (x, cos, sin, at + 6),
                 (x, cos[:0], sin[:0], at), (x, cos[:, :0], sin[:, :0])):
        with pytest.raises(ValueError):
            ops.rotary(*args)
    qkv, w = torch.randn(6, 2, 5 * 8), torch.ones(8)
    ops.qk_norm_rope(qkv, w, w, cos, sin, 3, 1)
    for args in ((qkv[0], w, w, cos, sin, 3, 1), (qkv, w, None, cos, sin, 3, 1), (qkv, w[:4], w, cos, sin, 3, 1),
                 (qkv, w.double(), w.double(), cos, sin, 3, 1), (qkv, w, w, cos, sin, 4, 1), (qkv, w, w, cos, sin, 0, 0),
                 (qkv, w, w, cos, sin, -1, 3), (qkv, w, w, cos, sin, 3, 1, -1e-5), (qkv, w, w, cos, sin, 3, 1, float("nan"))):
        with pytest.raises(ValueError):
            ops.qk_norm_rope(*args)
