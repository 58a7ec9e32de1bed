"""Masked attention (csrc/masked_attention*.cu) against 64 bits, and its mask against its definition.

Tolerances, derived beforehand. u = 2^-8 is half a step of bf16. Probabilities are rounded to bf16 before they meet v or
dO (u, relative), a result is rounded once more (u of the result), and what fp32 does before that (dot products of up to 128
terms with scores up to ~ 60, the exponential, the capped score to ~ 2^-18) changes a probability by less than f = 2^-12, relative:

  |dout|  <= u |out| + (u + f) p |v| + u |out|                         =: u |out| + A
             (out = sum_j P_j v_j / sum_j P_j of the rounded P_j = p_j (1 + e_j), |e_j| <= u: off by sum_j p_j e_j (v_j - out), and
             sum_j p_j |v_j - out| <= p |v| + |out|, nearly reached where two keys are seen)
  |ddV|   <= u |dV| + (u + f) p' |dO|
  dvec    = rowsum(dO * out): off by E = |dO| (u |out| + A) (out is saved more precisely than it is rounded: less than this)
  |ddQ|   <= u |dQ| + scale ((u + f) |dS| + p g (E + 2^-14 (|dP| + |dvec|))) |k|      g: derivative of the capped score
  |ddK|   <= the same with the transposed matrix and |q|

plus 2^-100 for results that are zero.
"""
import math

import pytest
import torch

from gpt_from_scratch_b200 import ops
from gpt_from_scratch_b200.ops import _lib
from gpt_from_scratch_b200.ops.masked_attention import _layout, _scratch

pytestmark = pytest.mark.gpu
U, F = 2.0 ** -8, 2.0 ** -12


def bounds_and_values(q, k, v, dout, see, softcap, slopes, scale):
    """(out, dq, dk, dv) in 64 bits and how far bf16 results may be from them. The formulas, written out."""
    q, k, v, do = (t.detach().double() for t in (q, k, v, dout))
    nh, nkv, S = q.shape[1], k.shape[1], q.shape[2]
    kk, vv = (t.repeat_interleave(nh // nkv, dim=1) for t in (k, v))
    s = q @ kk.transpose(-1, -2) * scale
    g = torch.ones_like(s)
    if softcap:
        t = torch.tanh(s / softcap)
        s, g = softcap * t, 1 - t * t
    if slopes is not None:
        at = torch.arange(S, device=q.device)
        s = s - slopes.double()[:, None, None] * (at[:, None] - at).abs()
    see = see.unsqueeze(1)
    s = s.masked_fill(~see, -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(-1e300)
    p = torch.exp(s - top)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    out = p @ vv
    A = (U + F) * (p @ vv.abs()) + U * out.abs()
    tol_out = U * out.abs() + A
    dP = do @ vv.transpose(-1, -2)
    dvec = (do * out).sum(-1, keepdim=True)
    dS = p * g * (dP - dvec)
    E = (do.abs() * tol_out).sum(-1, keepdim=True)
    err = (U + F) * dS.abs() + p * g * (E + 2.0 ** -14 * (dP.abs() + dvec.abs()))

    def shared(t):
        return t.unflatten(1, (nkv, nh // nkv)).sum(2)
    dq, dk, dv = scale * dS @ kk, shared(scale * dS.transpose(-1, -2) @ q), shared(p.transpose(-1, -2) @ do)
    tols = [tol_out, U * dq.abs() + scale * err @ kk.abs(), U * dk.abs() + shared(scale * err.transpose(-1, -2) @ q.abs()),
            U * dv.abs() + (U + F) * shared(p.transpose(-1, -2) @ do.abs())]
    return [out, dq, dk, dv], [t + 2.0 ** -100 for t in tols]


def check(got, want, tols, what=""):
    for a, b, tol, name in zip(got, want, tols, ("out", "dq", "dk", "dv")):
        assert a.dtype == torch.bfloat16 and a.shape == b.shape
        off = (a.double() - b).abs() / tol
        assert torch.isfinite(a).all(), f"{what} {name}: not finite"
        assert off.max() <= 1, f"{what} {name}: {off.max().item():.3g} of the bound, at {(off == off.max()).nonzero()[0].tolist()}"


def run(q, k, v, dout, mask, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.masked_attention(*leaves, mask, **kw)
    return [out.detach(), *torch.autograd.grad(out, leaves, dout)]


def document_ids(B, S, kind, seed):
    """none | docs: documents of 1 to S / 2 tokens | padded: some of them, and the end, padding | empty: one sequence all padding."""
    if kind == "none":
        return None
    g = torch.Generator().manual_seed(seed)
    rows = []
    for b in range(B):
        row, i = [], 0
        while len(row) < S:
            n = int(torch.randint(1, max(2, S // 2), (1,), generator=g))
            row += [-1 if kind == "padded" and i % 3 == 2 else i] * n
            i += 1
        row = row[:S]
        if kind != "docs" and S > 3:
            row[-(S // 4):] = [-1] * (S // 4)
        if kind == "empty" and b == 0:
            row = [-1] * S
        rows.append(row)
    return torch.tensor(rows, device="cuda")


@pytest.mark.parametrize("B,S", [(1, 1), (3, 2), (2, 127), (2, 128), (1, 129), (2, 1023), (2, 1025), (1, 2304), (1, 5001), (2, 17003)])
@pytest.mark.parametrize("kind", ["none", "docs", "padded", "empty"])
def test_mask(cuda_device, B, S, kind):
    ids = document_ids(B, S, kind, S)
    g = torch.Generator().manual_seed(S)
    prefix = (torch.rand(B, S, generator=g) < 0.95).to(cuda_device)
    for causal, pre, window in ((True, None, None), (False, None, None), (True, prefix, None), (True, None, 5), (True, prefix, 70),
                                (True, None, S), (True, None, 1), (True, None, 2 ** 40)):
        for typ in (torch.int64, torch.int32):
            at = None if ids is None else ids.to(typ)
            mask = ops.attention_mask(B, S, causal, at, pre, window, device=cuda_device)
            cpu = ops.attention_mask(B, S, causal, None if at is None else at.cpu(), None if pre is None else pre.cpu(), window)
            for name in ("first", "last", "positions"):
                assert torch.equal(getattr(mask, name).cpu(), getattr(cpu, name)), f"{name} {causal} {window}"
        # the queries of every key, as the backward reads them
        S_pad = (S + 127) // 128 * 128
        tiles = S_pad // 128
        layout = _layout(B, S)
        assert mask.buffer.numel() == layout["end"]
        qfirst, qlast, padded, plan_q, plan_k = (
            mask.buffer[layout[name]:layout[name] + math.prod(shape)].view(shape).cpu()
            for name, shape in (("qfirst", (B, S_pad)), ("qlast", (B, S_pad)), ("padded", (B,)), ("plan_q", (B, tiles, 4)),
                                ("plan_k", (B, tiles, 4))))
        # (by their first and last: both ends grow, so a query sees j from the first whose last is past j to the last whose first is not)
        at = torch.arange(S).expand(B, S).contiguous()
        lo = torch.searchsorted(cpu.last.long().contiguous(), at, right=True)
        hi = torch.searchsorted(cpu.first.long().contiguous(), at, right=True)
        j_any = torch.zeros(B, S, dtype=torch.bool) | (ids >= 0).cpu() if ids is not None else torch.ones(B, S, dtype=torch.bool)
        # queries that are padding see nothing and may lie in front of the first or behind the last
        if S <= 2500:
            see = cpu.visible()
            rows = torch.arange(S)[None, :, None]
            assert torch.equal(j_any, see.any(1))
            lo, hi = torch.where(see, rows, S).amin(1), torch.where(see, rows + 1, 0).amax(1)
        elif kind in ("padded", "empty"):
            lo, hi = qfirst[:, :S], qlast[:, :S]
        assert torch.equal(torch.where(j_any, qfirst[:, :S], 0), torch.where(j_any, lo, 0).int())
        assert torch.equal(torch.where(j_any, qlast[:, :S], 0), torch.where(j_any, hi, 0).int())
        assert (qfirst[:, :S][~j_any] == qlast[:, :S][~j_any]).all() and (qfirst[:, S:] == S).all() and (qlast[:, S:] == S).all()
        assert (qfirst.diff(dim=1) >= 0).all() and (qlast.diff(dim=1) >= 0).all()
        assert padded.bool().tolist() == ([False] * B if ids is None else (ids < 0).any(1).tolist())
        # the order of the tiles: every one once, with the ends of what it sees, the widest first
        ends = torch.arange(tiles) * 128, (torch.arange(tiles) * 128 + 127).clamp_max(S - 1)
        for plan, lo, hi in ((plan_q, cpu.first, cpu.last), (plan_k, qfirst, qlast)):
            for b in range(B):
                t = plan[b, :, 0].long()
                assert t.sort().values.tolist() == list(range(tiles))
                assert torch.equal(plan[b, :, 1], lo[b][ends[0][t]]) and torch.equal(plan[b, :, 2], hi[b][ends[1][t]])
                assert ((plan[b, :, 2] - plan[b, :, 1]).diff() <= 0).all()


#   B, nh, nkv, S, D, documents, causal, prefix, window, cap, distance
FORMS = [
    (1, 1, 1, 1, 64, "none", True, False, None, 0.0, False),
    (2, 2, 1, 1, 128, "none", True, False, None, 20.0, True),
    (1, 2, 2, 2, 64, "none", True, False, None, 0.0, False),
    (2, 4, 2, 127, 64, "docs", True, False, None, 0.0, False),
    (2, 4, 1, 128, 128, "docs", True, False, None, 0.0, False),
    (1, 3, 3, 129, 128, "none", True, False, None, 0.0, False),
    (2, 2, 2, 300, 64, "none", False, False, None, 0.0, False),
    (2, 2, 2, 300, 128, "docs", False, False, None, 0.0, True),
    (2, 6, 2, 333, 64, "docs", True, True, None, 0.0, False),
    (1, 6, 2, 640, 128, "docs", True, True, 200, 30.0, False),
    (2, 3, 1, 257, 128, "padded", True, False, None, 0.0, True),
    (3, 2, 2, 200, 64, "empty", True, False, None, 15.0, True),
    (2, 2, 1, 513, 64, "padded", True, True, 40, 0.0, False),
    (1, 2, 2, 700, 64, "none", True, False, 1, 0.0, False),
    (1, 2, 1, 700, 128, "none", True, False, 130, 50.0, False),
    (1, 8, 1, 1100, 64, "docs", True, False, None, 5.0, False),
    (1, 4, 4, 1100, 128, "none", True, False, None, 0.0, True),
    (8, 12, 12, 130, 64, "docs", True, False, None, 0.0, False),
    (1, 16, 16, 1500, 64, "padded", True, False, 300, 0.0, False),
    (2, 20, 4, 900, 128, "docs", True, True, None, 0.0, False),
    (1, 32, 8, 252, 128, "none", True, False, 2, 5.0, False),
]


def tensors(B, nh, nkv, S, D, seed, packed=True, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if packed:      # parts of the packed projection [S, B, heads, D]
        qkv = torch.randn(S, B, nh + 2 * nkv, D, device="cuda", generator=g).bfloat16()
        q, k, v = (t.permute(1, 2, 0, 3) for t in qkv.split([nh, nkv, nkv], 2))
    else:
        q, k, v = (torch.randn(B, n, S, D, device="cuda", generator=g).bfloat16() for n in (nh, nkv, nkv))
    return q * spread if not packed else q, k, v, torch.randn(B, nh, S, D, device="cuda", generator=g).bfloat16()


def build_mask(B, S, kind, causal, prefix, window):
    ids = document_ids(B, S, kind, S + B)
    g = torch.Generator().manual_seed(B * S)
    pre = (torch.rand(B, S, generator=g) < 0.97).cuda() if prefix else None
    return ops.attention_mask(B, S, causal, ids, pre, window, device="cuda"), ids


@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(str(x) for x in f))
def test_masked_attention(cuda_device, form):
    B, nh, nkv, S, D, kind, causal, prefix, window, cap, distance = form
    mask, _ = build_mask(B, S, kind, causal, prefix, window)
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / nh) for h in range(nh)], device=cuda_device) if distance else None
    for packed in (True, False):
        q, k, v, do = tensors(B, nh, nkv, S, D, S + D, packed)
        before = _lib.launch_count()
        out = ops.masked_attention(q, k, v, mask, softcap=cap, alibi_slopes=slopes)
        torch.cuda.synchronize()
        want, tols = bounds_and_values(q, k, v, do, mask.visible(), cap, slopes, 1 / math.sqrt(D))
        check([out], want, tols, "forward")
        got = run(q, k, v, do, mask, softcap=cap, alibi_slopes=slopes)
        assert _lib.launch_count() - before == 5 + (_scratch(S, B, nh, nkv, D) > 0)
        check(got, want, tols, f"packed {packed}")
        assert torch.equal(got[0], out)
        hidden = ~mask.visible().any(2)[:, None, :, None]
        assert (got[0].masked_select(hidden) == 0).all() and (got[1].masked_select(hidden) == 0).all()
        assert all((t.masked_select(hidden) == 0).all() for t in got[2:])


@pytest.mark.parametrize("D,cap", [(64, 0.0), (64, 20.0), (128, 0.0), (128, 20.0)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -3.0e38])
def test_padding_may_hold_anything(cuda_device, D, cap, what):
    B, nh, nkv, S = 2, 4, 2, 450
    mask, ids = build_mask(B, S, "padded", True, False, None)
    q, k, v, do = (t.clone() for t in tensors(B, nh, nkv, S, D, 5, packed=False))
    clean = run(q, k, v, do, mask, softcap=cap)
    pad = (ids < 0)[:, None, :, None]
    dirty = run(*(t.masked_fill(pad, what) for t in (q, k, v, do)), mask, softcap=cap)
    assert all(torch.equal(a, b) for a, b in zip(clean, dirty))


@pytest.mark.parametrize("D", [64, 128])
def test_growing_and_large_scores(cuda_device, D):
    """Keys that grow along the sequence raise the running maximum in every block; capped, they saturate both ways."""
    B, nh, S = 1, 2, 640
    q, k, v, do = tensors(B, nh, nh, S, D, 7, packed=False, spread=1.0)
    ramp = torch.linspace(0.1, 4.0, S, device=cuda_device)[:, None]
    k = (k.float() * ramp).bfloat16()
    mask = ops.attention_mask(B, S, device=cuda_device)
    for cap in (0.0, 2.0, 30.0):
        want, tols = bounds_and_values(q, k, v, do, mask.visible(), cap, None, 1 / math.sqrt(D))
        check(run(q, k, v, do, mask, softcap=cap), want, tols, f"cap {cap}")
    # explicit scale
    want, tols = bounds_and_values(q, k, v, do, mask.visible(), 0.0, None, 0.05)
    check(run(q, k, v, do, mask, scale=0.05), want, tols, "scale")


@pytest.mark.parametrize("cap", [0.0, 10.0, 50.0, 900.0])
def test_bias_that_grows_with_the_distance(cuda_device, cap):
    """Negative slopes: far keys win by hundreds, so a capped score plus its bias has no bound."""
    B, nh, S, D = 1, 3, 500, 64
    q, k, v, do = tensors(B, nh, nh, S, D, 13, packed=False)
    slopes = torch.tensor([-0.5, -2.0, 0.25], device=cuda_device)
    mask = ops.attention_mask(B, S, device=cuda_device)
    want, tols = bounds_and_values(q, k, v, do, mask.visible(), cap, slopes, 1 / 8)
    check(run(q, k, v, do, mask, softcap=cap, alibi_slopes=slopes), want, tols, f"cap {cap}")


def test_second_derivatives_are_refused(cuda_device):
    q, k, v, do = tensors(1, 2, 2, 40, 64, 1, packed=False)
    q = q.detach().requires_grad_()
    out = ops.masked_attention(q, k, v, ops.attention_mask(1, 40, device=cuda_device))
    dq, = torch.autograd.grad(out, q, do, create_graph=True)        # the first is computed as ever
    assert torch.equal(dq, run(q, k, v, do, ops.attention_mask(1, 40, device=cuda_device))[1])
    with pytest.raises(RuntimeError):
        dq.float().sum().backward()


def test_no_heads_and_gradients_of_some_inputs(cuda_device):
    mask = ops.attention_mask(2, 70, device=cuda_device)
    q, k, v, do = tensors(2, 4, 2, 70, 64, 1, packed=False)
    k = k.detach().requires_grad_()
    dk, = torch.autograd.grad(ops.masked_attention(q, k, v, mask), k, do)
    assert torch.equal(dk, run(q, k, v, do, mask)[2])
    dk, = torch.autograd.grad(ops.masked_attention(q[:, :0], k, v, mask), k, do[:, :0])
    assert (dk == 0).all()


def test_equals_causal_attention_of_the_framework(cuda_device):
    q, k, v, do = tensors(2, 3, 3, 512, 64, 3, packed=False)
    mask = ops.attention_mask(2, 512, device=cuda_device)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    ref = ops.apply_flash_attn(*leaves, True)
    ref_grads = torch.autograd.grad(ref, leaves, do)
    want, tols = bounds_and_values(q, k, v, do, mask.visible(), 0.0, None, 1 / 8)
    for a, b, tol in zip(run(q, k, v, do, mask), (ref.detach(), *ref_grads), tols):
        assert ((a.double() - b.double()).abs() <= 2 * tol).all()


def test_gradients_against_differences(cuda_device):
    """The forward in 64 bits, moved along a direction, against the kernel's gradients."""
    B, nh, nkv, S, D = 1, 4, 2, 90, 64
    mask, _ = build_mask(B, S, "docs", True, True, None)
    q, k, v, do = tensors(B, nh, nkv, S, D, 21, packed=False)
    slopes = torch.full((nh,), 0.1, device=cuda_device)
    grads = run(q, k, v, do, mask, softcap=10.0, alibi_slopes=slopes)[1:]
    _, tols = bounds_and_values(q, k, v, do, mask.visible(), 10.0, slopes, 1 / 8)
    args = [t.double() for t in (q, k, v)]
    step = 1e-4
    for i, grad in enumerate(grads):
        d = torch.randn(args[i].shape, dtype=torch.float64, device=cuda_device, generator=torch.Generator(device="cuda").manual_seed(i))

        def f(sign):
            moved = [t + (sign * step * d if j == i else 0) for j, t in enumerate(args)]
            return (ops.masked_attention_reference(*moved, mask, 10.0, slopes) * do.double()).sum().item()
        slope = (f(1) - f(-1)) / (2 * step)
        assert abs(slope - (grad.double() * d).sum().item()) <= (tols[1 + i] * d.abs()).sum().item() + 1e-4 * abs(slope)


def test_layouts_streams_and_graphs(cuda_device):
    B, nh, nkv, S, D = 2, 4, 2, 300, 64
    mask, ids = build_mask(B, S, "docs", True, False, None)
    q, k, v, do = tensors(B, nh, nkv, S, D, 2)
    want = run(q, k, v, do, mask, softcap=25.0)
    # misaligned, last dimension strided, broadcast over the batch: copied, same bits
    odd = torch.empty(q.numel() + 1, dtype=torch.bfloat16, device=cuda_device)[1:].view(q.shape).copy_(q)
    strided = torch.empty(*k.shape[:3], 2 * D, dtype=torch.bfloat16, device=cuda_device)[..., ::2].copy_(k)
    assert all(torch.equal(a, b) for a, b in zip(want, run(odd, strided, v, do, mask, softcap=25.0)))
    same = ops.attention_mask(B, S, document_ids=ids[:1].expand(B, S), device=cuda_device)
    shared = run(q[:1].expand_as(q), k[:1].expand_as(k), v[:1].expand_as(v), do[:1].expand_as(do), same)
    alone = run(q[:1], k[:1], v[:1], do[:1], ops.attention_mask(1, S, document_ids=ids[:1], device=cuda_device))
    assert all(torch.equal(a[b], c[0]) for a, c in zip(shared, alone) for b in range(B))
    # a scalar's gradient: dout is broadcast from one number
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    ops.masked_attention(*leaves, mask).sum().backward()
    ones = run(q, k, v, torch.ones_like(do), mask)
    assert all(torch.equal(t.grad, g) for t, g in zip(leaves, ones[1:]))
    # two streams at once
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for s in streams:
        with torch.cuda.stream(s):
            for _ in range(3):
                m = ops.attention_mask(B, S, document_ids=ids)
                results.append(run(q, k, v, do, m, softcap=25.0))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in results for a, b in zip(want, r))
    del results, leaves
    # captured, mask and all; replayed on other documents and other values
    static = [t.clone() for t in (q, k, v, do)]
    static_ids = ids.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m = ops.attention_mask(B, S, document_ids=static_ids)
        captured = run(*static, m, softcap=25.0)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, captured))
    static_ids.copy_(document_ids(B, S, "padded", 99))
    for t in static:
        t.copy_(t.flip(2))
    graph.replay()
    torch.cuda.synchronize()
    again = run(*static, ops.attention_mask(B, S, document_ids=static_ids), softcap=25.0)
    assert all(torch.equal(a, b) for a, b in zip(again, captured))


def test_empty_and_refused(cuda_device):
    for B, S in ((0, 5), (2, 0)):
        mask = ops.attention_mask(B, S, device=cuda_device)
        q = torch.empty(B, 4, S, 64, device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
        out = ops.masked_attention(q, q, q, mask)
        out.sum().backward()
        assert out.shape == q.shape == q.grad.shape
    mask = ops.attention_mask(1, 8, device=cuda_device)
    for t in (torch.randn(1, 2, 8, 64, device=cuda_device), torch.randn(1, 2, 8, 64, device=cuda_device).half(),
              torch.randn(1, 2, 8, 32, device=cuda_device).bfloat16()):
        with pytest.raises(ValueError):
            ops.masked_attention(t, t, t, mask)
    t = torch.randn(1, 2, 8, 64, device=cuda_device).bfloat16()
    with pytest.raises(ValueError):
        ops.masked_attention(t, t, t, ops.attention_mask(1, 8))      # a mask on the CPU
    for cap in (1e-9, 1e9):
        with pytest.raises(ValueError):
            ops.masked_attention(t, t, t, mask, softcap=cap)
    many = t[:, :, :1].expand(70000, 2, 1, 64)
    with pytest.raises(ValueError):
        ops.masked_attention(many, many, many, ops.attention_mask(70000, 1, device=cuda_device))
    with pytest.raises(ValueError):
        ops.attention_mask(1, 8, document_ids=torch.zeros(1, 8, dtype=torch.int32), device=cuda_device)


def test_positions_norm_rotation_and_attention_together(cuda_device):
    """A packed batch through mask -> qk_norm_rope -> masked_attention and back, against the same in 64 bits."""
    B, nh, nkv, S, D = 2, 4, 2, 260, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    ids = document_ids(B, S, "padded", 8)
    mask = ops.attention_mask(B, S, document_ids=ids)
    qkv = torch.randn(S, B, (nh + 2 * nkv) * D, device=cuda_device, generator=g).bfloat16()
    w = [(1 + 0.2 * torch.randn(D, device=cuda_device, generator=g)).bfloat16() for _ in range(2)]
    dout = torch.randn(S, B, nh * D, device=cuda_device, generator=g).bfloat16()
    cos, sin = ops.rope_tables(S, D, device=cuda_device)

    def block(qkv, wq, wk, norm, attend):
        q, k, v = norm(qkv, wq, wk, cos, sin, nh, nkv, positions=mask.positions)
        o = attend(*(t.permute(1, 2, 0, 3) for t in (q, k, v)), mask, softcap=20.0)
        return o.permute(2, 0, 1, 3).reshape(S, B, nh * D)

    def both(dtype, norm, attend):
        leaves = [t.detach().to(dtype).requires_grad_() for t in (qkv, *w)]
        out = block(*leaves, norm, attend)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout.to(dtype))]
    got = both(torch.bfloat16, ops.qk_norm_rope, ops.masked_attention)
    want = both(torch.float64, ops.qk_norm_rope_reference, ops.masked_attention_reference)
    # three roundings to bf16 in a row (q and k, p or dS, the result), each 2^-8 of its value at most and 2^-8 / sqrt(3) of it in the
    # root mean square; scores of size ~ 8 pass a relative error of q and k on as 8 sqrt(2 / D) of it: 2-norms within 2^-6
    for a, b in zip(got, want):
        assert torch.isfinite(a).all() and (a.double() - b).norm() <= 2.0 ** -6 * b.norm()
    pad = (ids < 0).t()
    assert (got[0][pad] == 0).all() and (got[1][pad] == 0).all()


@pytest.mark.parametrize("D", [64, 128])
def test_gradients_of_scores_do_not_see_the_rounding_of_outputs(cuda_device, D):
    """Documents of two tokens with one key twice and values a few steps apart: the second query's output lies between two bf16 numbers, and
    its gradients are what differs between the values."""
    B, H, S = 2, 2, 82
    gen = torch.Generator(device="cuda").manual_seed(D)
    q, k, dout = (torch.randn(B, H, S, D, device="cuda", generator=gen).bfloat16() for _ in range(3))
    k[:, :, 1::2] = k[:, :, 0::2]
    steps = torch.randint(1, 100, (B, H, S, D), device="cuda", generator=gen)
    steps[:, :, 1::2] = steps[:, :, 0::2] + torch.randint(-3, 4, (B, H, S // 2, D), device="cuda", generator=gen)
    v = (1.0 + steps * 2.0 ** -7).bfloat16()                       # in [1, 2), where a step is 2^-7
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    ids = (torch.arange(S, device="cuda") // 2).int().expand(B, S)
    out = ops.masked_attention(q, k, v, ops.attention_mask(B, S, document_ids=ids))
    dk, = torch.autograd.grad(out, k, dout)

    first, second = slice(0, None, 2), slice(1, None, 2)
    q64, v64, do64 = (t.detach().double() for t in (q, v, dout))
    ds = 0.25 * (do64[:, :, second] * (v64[:, :, first] - v64[:, :, second])).sum(-1, keepdim=True)
    want = torch.zeros_like(q64)
    want[:, :, first], want[:, :, second] = ds * q64[:, :, second] / D ** 0.5, -ds * q64[:, :, second] / D ** 0.5
    # dS and dk are rounded to bf16 once each, P = 1/2 is recomputed to less than 2^-15. dP - dvec, of which dS is half: outputs of 1 to 2
    # are saved to 2^-8 of a step of 2^-7 (2^-16 of `size`), and both are sums of D products in 32 bits
    size = (do64.abs() * 2.0).sum(-1, keepdim=True)
    off = 0.5 * size * (2.0 ** -16 + 2 * D * 2.0 ** -24)
    off = off[:, :, second] * q64[:, :, second].abs() / D ** 0.5
    bound = want.abs() * (2 * 2.0 ** -8 + 2.0 ** -15)
    for part in (first, second):
        bound[:, :, part] += off * (1 + 2 * 2.0 ** -8)
    # the first query sees its own key alone: dP - dvec is the sums' rounding
    bound[:, :, first] += size[:, :, first] * 2 * D * 2.0 ** -24 * q64[:, :, first].abs() / D ** 0.5
    assert ((dk.double() - want).abs() <= bound).all()


def test_offsets_past_32_bits(cuda_device):
    """2.25e9 numbers in q and all that is like it; the last queries and keys are looked at."""
    B, nh, S, D, window, tail = 1, 16, 1_100_000, 128, 64, 512
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, dout = (torch.empty(B, nh, S, D, device="cuda", dtype=torch.bfloat16).normal_(generator=gen) for _ in range(2))
    k, v = (torch.empty(B, 1, S, D, device="cuda", dtype=torch.bfloat16).normal_(generator=gen) for _ in range(2))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ops.masked_attention(*leaves, ops.attention_mask(B, S, window=window, device="cuda"))
    grads = torch.autograd.grad(out, leaves, dout)
    at = torch.arange(tail, device="cuda")
    see = ((at[:, None] >= at) & (at > at[:, None] - window)).expand(B, tail, tail)
    wants, tols = bounds_and_values(*(t[:, :, -tail:] for t in (q, k, v, dout)), see, 0.0, None, D ** -0.5)
    for got, want, tol in zip((out, *grads), wants, tols):       # (the tail's first queries see keys before it)
        assert ((got[:, :, -tail:].double() - want).abs() <= tol)[:, :, window:].all()
    del out, grads, dout

    x = q.detach().view(S, B, nh, D)
    cos, sin = ops.rope_tables(S, D, device="cuda")
    want = ops.rotary_reference(x[-tail:].double(), cos[-tail:].double(), sin[-tail:].double())
    off = (ops.rotary(x, cos, sin)[-tail:].double() - want).abs()
    assert (off <= U * want.abs() + 2.0 ** -22 * x[-tail:].double().abs().amax()).all()
