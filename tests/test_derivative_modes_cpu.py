"""What operators on raw pointers owe to autograd's other modes (ops/_lib.py: bare, first_order), with a function of that form."""
import warnings

import pytest
import torch
import torch.autograd.forward_ad as fwd

from gpt_from_scratch_b200.ops import _lib


class Double(torch.autograd.Function):
    """Writes through a pointer, unseen by autograd, like the kernels."""
    @staticmethod
    def forward(ctx, x):
        ctx.traced = torch._C._is_tracing()
        y = torch.empty_like(x)
        y.numpy()[:] = 2 * x.detach().numpy()
        return y

    @staticmethod
    @_lib.first_order
    def backward(ctx, dy):
        dx = torch.empty(dy.shape)
        dx.numpy()[:] = 2 * dy.detach().numpy()
        return dx


def test_when_the_function_may_be_left_out():
    x = torch.ones(3)
    assert _lib.bare(x, None)
    w = x.clone().requires_grad_()
    assert not _lib.bare(x, w)
    with torch.no_grad():
        assert _lib.bare(x, w)
        with fwd.dual_level():                  # forward mode does not ask for the grad mode
            assert not _lib.bare(fwd.make_dual(x, x))
    assert _lib.bare(x)
    seen = []
    torch.jit.trace(lambda t: (seen.append(_lib.bare(t)), t + 1)[1], (x,), check_trace=False)
    assert seen == [False]


def test_a_backward_refuses_tangents():
    x = torch.ones(3, requires_grad=True)
    with fwd.dual_level():
        y = Double.apply(x)
        dx, = torch.autograd.grad(y, x, torch.ones(3), retain_graph=True)      # none here
        assert torch.equal(dx, torch.full((3,), 2.0))
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(y, x, fwd.make_dual(torch.ones(3), torch.ones(3)))


def test_a_backward_is_not_traced():
    def f(x):
        x = x.detach().requires_grad_()
        return torch.autograd.grad(Double.apply(x).sum(), x)[0]
    with warnings.catch_warnings(), pytest.raises(NotImplementedError):
        warnings.simplefilter("ignore")
        torch.jit.trace(f, (torch.ones(3),), check_trace=False)
