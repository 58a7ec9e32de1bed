"""Forward-mode derivatives, traces and the operators of the attention block: refused or right, never without the derivative or with
an output that nothing wrote."""
import warnings

import pytest
import torch
import torch.autograd.forward_ad as fwd

from gpt_from_scratch_b200 import ops

pytestmark = pytest.mark.gpu

S, B, NH, NKV, D = 70, 2, 4, 2, 64


def operators(device):
    """name -> (call on its floating-point inputs, the inputs)"""
    gen = torch.Generator(device=device).manual_seed(0)

    def normal(*shape):
        return torch.randn(*shape, device=device, generator=gen).bfloat16()
    cos, sin = ops.rope_tables(S, D, device=device)
    ids = (torch.arange(S, device=device) // 30).expand(B, S)
    mask = ops.attention_mask(B, S, document_ids=ids)
    return {
        "rotary": (lambda x: ops.rotary(x, cos, sin), [normal(S, B, NH, D)]),
        "qk_norm_rope": (lambda x, a, b: torch.cat(ops.qk_norm_rope(x, a, b, cos, sin, NH, NKV, positions=mask.positions), dim=2),
                         [normal(S, B, (NH + 2 * NKV) * D), normal(D), normal(D)]),
        "masked_attention": (lambda q, k, v: ops.masked_attention(q, k, v, mask, softcap=20.0),
                             [normal(B, NH, S, D), normal(B, NKV, S, D), normal(B, NKV, S, D)]),
    }


NAMES = ["rotary", "qk_norm_rope", "masked_attention"]


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(cuda_device, name, grad):
    call, inputs = operators(cuda_device)[name]
    for i in range(len(inputs)):
        with fwd.dual_level(), torch.set_grad_enabled(grad):
            args = [fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(inputs)]
            with pytest.raises(NotImplementedError):
                call(*args)
    with fwd.dual_level():                      # an open level by itself changes nothing
        inside = call(*inputs)
    assert torch.equal(inside, call(*inputs))


@pytest.mark.parametrize("name", NAMES)
def test_tangents_of_gradients_are_refused(cuda_device, name):
    call, inputs = operators(cuda_device)[name]
    leaves = [t.requires_grad_() for t in inputs]
    out = call(*leaves)
    with fwd.dual_level(), pytest.raises(NotImplementedError):
        torch.autograd.grad(out, leaves, fwd.make_dual(torch.ones_like(out), torch.ones_like(out)))


def trace(f, *args):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        return torch.jit.trace(f, args, check_trace=False)


@pytest.mark.parametrize("name", NAMES)
def test_a_trace_calls_the_kernel_again(cuda_device, name):
    call, inputs = operators(cuda_device)[name]
    traced = trace(lambda *a: call(*a), *inputs)
    others = [t.flip(0) * 0.5 for t in inputs]
    assert torch.equal(traced(*others), call(*others)) and not torch.equal(call(*others), call(*inputs))
    leaves = [t.requires_grad_() for t in inputs]      # weights ask for gradients, and a traced forward gives them
    traced = trace(lambda *a: call(*a), *leaves)
    others = [t.detach().requires_grad_() for t in others]
    out = call(*others)
    dout = torch.ones_like(out)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(traced(*others), others, dout),
                                                 torch.autograd.grad(out, others, dout)))


def test_a_trace_makes_its_mask_again(cuda_device):
    q, k, v = operators(cuda_device)["masked_attention"][1]

    def f(q, k, v, ids):
        return ops.masked_attention(q, k, v, ops.attention_mask(B, S, document_ids=ids))
    ids, other = ((torch.arange(S, device=cuda_device) // n).expand(B, S).contiguous() for n in (30, 11))
    traced = trace(f, q, k, v, ids)
    assert torch.equal(traced(q, k, v, other), f(q, k, v, other)) and not torch.equal(f(q, k, v, other), f(q, k, v, ids))


@pytest.mark.parametrize("name", NAMES)
def test_a_traced_backward_is_refused(cuda_device, name):
    call, inputs = operators(cuda_device)[name]

    def gradient(*args):
        leaves = [t.detach().requires_grad_() for t in args]
        return torch.autograd.grad(call(*leaves).float().sum(), leaves)
    with pytest.raises(NotImplementedError):
        trace(gradient, *inputs)
