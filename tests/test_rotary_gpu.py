"""Rotary positions and the norms of q and k (csrc/rotary.cu) against 64 bits.

Tolerances, derived beforehand: a result is rounded once, to within eps / 2 of its type, relative (float16 results
below 2^-14: 2^-25 absolute). What comes before is fp32: a rotation has two products and a sum of numbers up to M
(the largest of the row), off by at most 3 * 2^-24 * 2 M; the norm's factor comes from a sum of D squares (positive: relative error
at most D 2^-24, 2^-16 for D = 256, halved by the root) and rsqrt (2 ulp), and the backward's mean of D products likewise, relative
to the sum of their magnitudes, so 2^-15 of the row's scale covers a row. Weight gradients are sums of N terms, each off like that,
added in fp32 in chains of far fewer than 2^9 (a thread's rows) + 2^6: 2^-14 of the sum of magnitudes.
"""
import pytest
import torch

from gpt_from_scratch_b200 import ops
from gpt_from_scratch_b200.ops import _lib

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def check(got, want, scale, slack, what):
    """|got - want| <= half a step of got's type + slack * scale (a tensor that broadcasts, in 64 bits)."""
    assert got.shape == want.shape, what
    half = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    off = (got.double() - want).abs() - half * want.abs() - tiny - slack * scale
    assert torch.isfinite(got).all() and (off <= 0).all(), f"{what}: {off.max().item():.3g} past the bound"


def inputs(S, B, n, D, dtype, seed, strided=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if strided:      # every second head of a wider tensor, batch first
        return torch.randn(B, S, 2 * n, D, device="cuda", generator=g).to(dtype)[:, :, ::2].transpose(0, 1)
    return torch.randn(S, B, n, D, device="cuda", generator=g).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("S,B,n,D,R", [(1, 1, 1, 64, 64), (5, 3, 7, 64, 32), (130, 2, 5, 128, 128), (33, 1, 4, 128, 32),
                                       (17, 2, 3, 256, 256), (9, 2, 3, 80, 80), (9, 2, 3, 80, 20), (7, 1, 2, 96, 96),
                                       (4, 2, 3, 34, 14), (3, 2, 1, 2, 2), (777, 2, 3, 64, 64)])
def test_rotary(cuda_device, S, B, n, D, R, interleaved, dtype):
    x = inputs(S, B, n, D, dtype, S * D + R, strided=S % 2 == 1).requires_grad_()
    dy = inputs(S, B, n, D, dtype, S * D + R + 1)
    cos, sin = ops.rope_tables(S + 50, R, device=cuda_device)
    g = torch.Generator(device="cuda").manual_seed(3)
    positions = torch.randint(0, S + 50, (B, S), device=cuda_device, generator=g)
    for at in (None, positions, positions.int()):
        before = _lib.launch_count()
        y = ops.rotary(x, cos, sin, at, interleaved)
        dx, = torch.autograd.grad(y, x, dy)
        assert _lib.launch_count() - before == 2 and y.dtype == dx.dtype == dtype
        x64 = x.detach().double().requires_grad_()
        want = ops.rotary_reference(x64, cos, sin, at, interleaved)
        dwant, = torch.autograd.grad(want, x64, dy.double())
        for got, ref, src, what in ((y, want, x, "y"), (dx, dwant, dy, "dx")):
            check(got, ref, src.detach().double().abs().amax(-1, keepdim=True), 6 * 2.0 ** -24, f"{what} {at is None}")
        if R < D:
            assert torch.equal(y[..., R:], x[..., R:]) and torch.equal(dx[..., R:], dy[..., R:])


def test_rotary_gradient_against_differences(cuda_device):
    cos, sin = ops.rope_tables(6, 8, device=cuda_device)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(6, 1, 2, 16, device=cuda_device, generator=g, requires_grad=True)
    dy = torch.randn(6, 1, 2, 16, device=cuda_device, generator=g)
    dx, = torch.autograd.grad(ops.rotary(x, cos, sin, interleaved=False), x, dy)
    v = torch.randn(6, 1, 2, 16, device=cuda_device, generator=g)
    with torch.no_grad():   # linear: the difference is exact but for rounding
        diff = ((ops.rotary(x + v, cos, sin, interleaved=False) - ops.rotary(x - v, cos, sin, interleaved=False)) / 2 * dy).sum()
    assert abs(diff.item() - (dx * v).sum().item()) < 192 * 8 * 2.0 ** -24 * 16


def test_rotary_matches_the_models_rotation(cuda_device):
    """The whole head, pairs side by side: what apply_rope computes, bit for bit."""
    x = inputs(64, 2, 3, 64, torch.bfloat16, 9)
    cos, sin = ops.rope_tables(64, 64, device=cuda_device)
    assert torch.equal(ops.rotary(x, cos, sin), ops.apply_rope(x, cos, sin))


def test_misaligned_and_empty(cuda_device):
    cos, sin = ops.rope_tables(5, 64, device=cuda_device)
    flat = torch.randn(5 * 2 * 3 * 64 + 1, device=cuda_device).bfloat16()
    x = flat[1:].view(5, 2, 3, 64)          # two bytes off any 16-byte boundary
    assert torch.equal(ops.rotary(x, cos, sin), ops.rotary(x.clone(), cos, sin))
    assert ops.rotary(torch.empty(0, 2, 3, 64, device=cuda_device).bfloat16(), cos, sin).shape == (0, 2, 3, 64)
    w = torch.ones(64, device=cuda_device).bfloat16()
    qkv = torch.empty(0, 2, 5 * 64, device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    w.requires_grad_()
    q, k, v = ops.qk_norm_rope(qkv, w, w, cos, sin, 3, 1)
    (q.sum() + k.sum() + v.sum()).backward()
    assert q.shape == (0, 2, 3, 64) and (w.grad == 0).all()


@pytest.mark.expects_status
def test_position_outside_of_the_tables_is_reported(cuda_device):
    cos, sin = ops.rope_tables(4, 64, device=cuda_device)
    x = inputs(3, 1, 2, 64, torch.bfloat16, 1)
    _lib.read_status(clear=True)
    ops.rotary(x, cos, sin, torch.tensor([[0, 4, -1]], device=cuda_device))     # the kernel clamps and reports them
    with pytest.raises(_lib.NativeLibraryError):
        _lib.raise_on_status()
    ops.rotary(x, cos, sin, torch.tensor([[0, 3, 1]], device=cuda_device))
    _lib.raise_on_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,B,n1,n2,D,R,interleaved,norm", [
    (1, 1, 1, 1, 64, 64, True, True), (130, 1, 12, 12, 64, 64, True, True), (33, 3, 6, 2, 128, 128, False, True),
    (7, 2, 5, 1, 128, 64, False, True), (40, 2, 4, 4, 256, 256, True, True), (11, 2, 3, 1, 80, 80, False, True),
    (6, 2, 3, 2, 34, 14, False, True), (6, 2, 3, 2, 34, 14, True, True), (300, 4, 8, 2, 96, 48, False, True),
    (50, 2, 4, 2, 64, 64, True, False), (9, 1, 3, 1, 70, 70, False, False)])
def test_qk_norm_rope(cuda_device, S, B, n1, n2, D, R, interleaved, norm, dtype):
    g = torch.Generator(device="cuda").manual_seed(S + D)
    wide = torch.randn(S, B, (n1 + 2 * n2) * D + 8, device=cuda_device, generator=g).to(dtype) * 1.5
    qkv = wide[..., 8:] if S % 2 else wide[..., 8:].contiguous()
    qkv[0, 0, :D] = 0                                   # a head of zeros: only eps keeps it finite
    w = [(1 + 0.3 * torch.randn(D, device=cuda_device, generator=g)).to(dtype) for _ in range(2)] if norm else [None] * 2
    # gradients of q in the layout that attention leaves them in
    dq = torch.randn(B, n1, S, D, device=cuda_device, generator=g).to(dtype).permute(2, 0, 1, 3)
    dk, dv = (torch.randn(S, B, n2, D, device=cuda_device, generator=g).to(dtype) for _ in range(2))
    cos, sin = ops.rope_tables(S + 9, R, device=cuda_device)
    positions = torch.randint(0, S + 9, (B, S), device=cuda_device, generator=g, dtype=torch.int32)
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (qkv, *w)]
    q, k, v = ops.qk_norm_rope(*leaves, cos, sin, n1, n2, eps=1e-5, positions=positions, interleaved=interleaved)
    assert torch.equal(v, qkv.unflatten(-1, (-1, D))[:, :, n1 + n2:])
    wrt = [t for t in leaves if t is not None]
    grads = torch.autograd.grad((q, k, v), wrt, (dq, dk, dv))
    wide_leaves = [t.detach().double().requires_grad_() if t is not None else None for t in leaves]
    q6, k6, v6 = ops.qk_norm_rope_reference(*wide_leaves, cos, sin, n1, n2, 1e-5, positions, interleaved)
    want = torch.autograd.grad((q6, k6, v6), [t for t in wide_leaves if t is not None], [t.double() for t in (dq, dk, dv)])
    slack = 2.0 ** -15
    for got, ref, what in ((q, q6, "q"), (k, k6, "k")):
        check(got, ref.detach(), ref.detach().abs().amax(-1, keepdim=True) * 2, slack, what)
    # the scale of a row's gradient: rstd * |dy| * |w|, for the term itself and for the mean it loses
    x = qkv.detach().double().unflatten(-1, (-1, D))
    rstd = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) if norm else torch.ones_like(x[..., :1])
    dy = torch.cat((dq, dk, dv), 2).double()
    wmax = max(float(t.detach().abs().max()) for t in w) if norm else 1.0
    xn = (x * rstd).abs()
    per_row = rstd * dy.abs().amax(-1, keepdim=True) * 2 * wmax * (1 + xn.amax(-1, keepdim=True) * xn.mean(-1, keepdim=True))
    check(grads[0].unflatten(-1, (-1, D)), want[0].unflatten(-1, (-1, D)), per_row, slack, "dqkv")
    assert torch.equal(grads[0].unflatten(-1, (-1, D))[:, :, n1 + n2:], dv)
    if norm:
        for i, (a, b) in enumerate(((0, n1), (n1, n1 + n2))):
            total = (dy[:, :, a:b].abs().amax(-1, keepdim=True) * 2 * xn[:, :, a:b]).sum((0, 1, 2))
            check(grads[1 + i], want[1 + i], total, 2.0 ** -14, f"dw{i}")


def test_qk_norm_rope_gradient_against_differences(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(8)
    cos, sin = ops.rope_tables(5, 64, device=cuda_device)
    qkv = torch.randn(5, 2, 4 * 64, device=cuda_device, generator=g)
    w = [1 + 0.2 * torch.randn(64, device=cuda_device, generator=g) for _ in range(2)]
    dq, dk = torch.randn(5, 2, 2, 64, device=cuda_device, generator=g), torch.randn(5, 2, 1, 64, device=cuda_device, generator=g)

    def f(x, a, b):
        q, k, _ = ops.qk_norm_rope(x, a, b, cos, sin, 2, 1)
        return (q.double() * dq).sum().item() + (k.double() * dk).sum().item()
    leaves = [t.clone().requires_grad_() for t in (qkv, *w)]
    q, k, _ = ops.qk_norm_rope(*leaves, cos, sin, 2, 1)
    grads = torch.autograd.grad((q, k), leaves, (dq, dk))
    step = 2.0 ** -7
    for i, grad in enumerate(grads):
        v = torch.randn(grad.shape, device=cuda_device, generator=g)
        moved = [[t + (sign * step * v if j == i else 0) for j, t in enumerate((qkv, *w))] for sign in (1, -1)]
        slope = (f(*moved[0]) - f(*moved[1])) / (2 * step)
        # central differences: O(step^2) of the third derivative, and the rounding of 1,920 terms of size ~1 over 2 step
        size = (grad.double() * v).abs().sum().item()
        assert abs(slope - (grad.double() * v).sum().item()) < (step * step * 20 + 2.0 ** -12) * size


def test_other_stream_graph_and_determinism(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(2)
    cos, sin = ops.rope_tables(200, 64, device=cuda_device)
    qkv = torch.randn(200, 3, 8 * 64, device=cuda_device, generator=g).bfloat16().requires_grad_()
    w = [torch.ones(64, device=cuda_device).bfloat16().requires_grad_() for _ in range(2)]
    grads_in = [torch.randn(200, 3, n, 64, device=cuda_device, generator=g).bfloat16() for n in (4, 2, 2)]

    def step():
        outs = ops.qk_norm_rope(qkv, *w, cos, sin, 4, 2)
        return [*(o.detach() for o in outs), *torch.autograd.grad(outs, (qkv, *w), grads_in)]
    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    del again
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for t in captured:
        t.zero_() if t._base is None else None
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, captured))
