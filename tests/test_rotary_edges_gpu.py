"""Norms of q and k at the edges of their arguments (csrc/rotary.cu), against 64 bits. Tolerances: those of test_rotary_gpu.py, whose
derivation covers eps = 0 as long as no row is all zeros."""
import pytest
import torch
from test_rotary_gpu import TYPES, check

from gpt_from_scratch_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n1,n2", [(1, 1), (3, 1), (5, 3), (4, 4)])
def test_norms_without_eps(cuda_device, n1, n2, D, dtype):
    """Head counts that leave groups of lanes without a head."""
    S, B = 9, 2
    gen = torch.Generator(device=cuda_device).manual_seed(n1 * D)

    def normal(*shape):
        return torch.randn(*shape, device=cuda_device, generator=gen).to(dtype)
    leaves = [normal(S, B, (n1 + 2 * n2) * D).requires_grad_(), *((1 + 0.3 * normal(D)).requires_grad_() for _ in range(2))]
    douts = [normal(S, B, n, D) for n in (n1, n2, n2)]
    cos, sin = ops.rope_tables(S, D, device=cuda_device)
    outs = ops.qk_norm_rope(*leaves, cos, sin, n1, n2, eps=0.0)
    grads = torch.autograd.grad(outs, leaves, douts)
    leaves6 = [t.detach().double().requires_grad_() for t in leaves]
    outs6 = ops.qk_norm_rope_reference(*leaves6, cos, sin, n1, n2, 0.0)
    wants = torch.autograd.grad(outs6, leaves6, [t.double() for t in douts])
    for got, want in zip(outs[:2], outs6[:2]):
        check(got, want.detach(), want.detach().abs().amax(-1, keepdim=True) * 2, 2.0 ** -15, "out")
    x = leaves6[0].detach().unflatten(-1, (-1, D))
    rstd = torch.rsqrt(x.square().mean(-1, keepdim=True))
    xn = (x * rstd).abs()
    dy = torch.cat(douts, 2).double()
    wmax = max(float(t.detach().abs().max()) for t in leaves[1:])
    per_row = rstd * dy.abs().amax(-1, keepdim=True) * 2 * wmax * (1 + xn.amax(-1, keepdim=True) * xn.mean(-1, keepdim=True))
    check(grads[0].unflatten(-1, (-1, D)), wants[0].unflatten(-1, (-1, D)), per_row, 2.0 ** -15, "dqkv")
    for i, (a, b) in enumerate(((0, n1), (n1, n1 + n2))):
        total = (dy[:, :, a:b].abs().amax(-1, keepdim=True) * 2 * xn[:, :, a:b]).sum((0, 1, 2))
        check(grads[1 + i], wants[1 + i], total, 2.0 ** -14, f"dw{i}")
