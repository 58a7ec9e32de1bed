"""The operators of the attention block called from several threads, replayed from several graphs, and past 32-bit offsets."""
import threading

import pytest
import torch
from test_rotary_gpu import check

from gpt_from_scratch_b200 import ops

pytestmark = pytest.mark.gpu


def block(seed, S=300, B=2, nh=4, nkv=2, D=64):
    """A function that runs mask, norms with rotation, attention and their gradients on inputs of its own."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(S, B, (nh + 2 * nkv) * D, device="cuda", generator=gen).bfloat16().requires_grad_()
    w = [torch.randn(D, device="cuda", generator=gen).bfloat16().requires_grad_() for _ in range(2)]
    dout = torch.randn(B, nh, S, D, device="cuda", generator=gen).bfloat16()
    ids = (torch.arange(S, device="cuda") // (40 + seed)).expand(B, S).contiguous()
    cos, sin = ops.rope_tables(S, D, device="cuda")

    def run():
        mask = ops.attention_mask(B, S, document_ids=ids)
        q, k, v = ops.qk_norm_rope(qkv, *w, cos, sin, nh, nkv, positions=mask.positions)
        out = ops.masked_attention(*(t.permute(1, 2, 0, 3) for t in (q, k, v)), mask, softcap=20.0)
        return [out.detach(), *torch.autograd.grad(out, (qkv, *w), dout)]
    return run


def test_threads(cuda_device):
    """Each with a stream and inputs of its own."""
    runs = [block(seed) for seed in range(4)]
    wants = [run() for run in runs]
    torch.cuda.synchronize()
    results = [[] for _ in runs]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(8):
                results[i].append(runs[i]())
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(runs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for want, got in zip(wants, results):
        assert len(got) == 8 and all(torch.equal(a, b) for one in got for a, b in zip(want, one))


def test_graphs_replayed_beside_each_other(cuda_device):
    """Workspaces belong to a call, so to a graph."""
    runs = [block(seed) for seed in range(2)]
    wants = [run() for run in runs]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in runs]
    for run in runs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run())
    for _ in range(10):
        for got in outs:
            for t in got:
                t.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for want, got in zip(wants, outs) for a, b in zip(want, got))


def test_norms_past_32_bit_offsets(cuda_device):
    """2.3e9 numbers in the projection; the last tokens are looked at. Tolerances: those of test_rotary_gpu.py."""
    S, nh, nkv, D, tail = 1_000_000, 16, 1, 128, 64
    gen = torch.Generator(device="cuda").manual_seed(0)

    def normal(*shape):
        return torch.empty(*shape, device="cuda", dtype=torch.bfloat16).normal_(generator=gen)
    qkv = normal(S, 1, (nh + 2 * nkv) * D).requires_grad_()
    w = [(1 + 0.25 * normal(D)).requires_grad_() for _ in range(2)]
    douts = [normal(S, 1, n, D) for n in (nh, nkv, nkv)]
    cos, sin = ops.rope_tables(S, D, device="cuda")
    outs = ops.qk_norm_rope(qkv, *w, cos, sin, nh, nkv)
    dqkv, = torch.autograd.grad(outs, qkv, douts)
    leaves = [t.detach().double().requires_grad_() for t in (qkv[-tail:], *w)]
    at = torch.arange(S - tail, S, device="cuda").expand(1, tail)
    wants = ops.qk_norm_rope_reference(*leaves, cos, sin, nh, nkv, 1e-5, at)
    dwant, = torch.autograd.grad(wants, leaves[0], [t[-tail:].double() for t in douts])
    for got, want in zip(outs[:2], wants[:2]):
        check(got[-tail:], want.detach(), want.detach().abs().amax(-1, keepdim=True) * 2, 2.0 ** -15, "out")
    x = leaves[0].detach().unflatten(-1, (-1, D))
    rstd = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)
    xn = (x * rstd).abs()
    wmax = max(float(t.detach().abs().max()) for t in w)
    dy = torch.cat([t[-tail:] for t in douts], 2).double().abs().amax(-1, keepdim=True)
    per_row = rstd * dy * 2 * wmax * (1 + xn.amax(-1, keepdim=True) * xn.mean(-1, keepdim=True))
    check(dqkv[-tail:].unflatten(-1, (-1, D)), dwant.unflatten(-1, (-1, D)), per_row, 2.0 ** -15, "dqkv")
