"""Training with norms of q and k, capped scores, a window and documents on the GPU.

Tolerance, derived beforehand: the fused and the eager path round the same values to bf16, each rounding off by 2^-8 / sqrt(3) of
the value in the root mean square; about a dozen in a row per block and direction, two blocks, both directions, two paths that differ
independently: sqrt(2 * 48) * 2^-8 / sqrt(3) = 0.022 of a 2-norm; 2^-5 covers it.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

CFG = dict(vocab_size=1024, num_layers=2, max_position_embeddings=512, intermediate_size=512, qk_norm=True, attention_softcap=20.0,
           attention_window=150, eod_token_id=0)


def engine(impl, graph=False, **cfg):
    from gpt_from_scratch_b200.config import GPTConfig
    from gpt_from_scratch_b200.engine import TrainEngine
    from gpt_from_scratch_b200.parallel import parallel_state as ps
    ps.set_device(torch.device("cuda", 0))
    ps.initialize_parallel_state(1)
    return TrainEngine(GPTConfig(**{**CFG, **cfg}, attention_impl=impl), lr=1e-3, seed=7, cuda_graph=graph)


def batch(step, B=2, S=260):
    g = torch.Generator().manual_seed(step)
    t = torch.randint(1, 1024, (B, S + 1), generator=g)
    t[torch.rand(B, S + 1, generator=g) < 0.01] = 0
    t = t.cuda()
    return t[:, :-1].contiguous(), t[:, 1:].contiguous()


@pytest.mark.parametrize("hidden,heads", [(256, 4), (256, 2)])
def test_fused_and_eager_attention_train_alike(cuda_device, hidden, heads):
    from gpt_from_scratch_b200.ops import _lib
    grads = {}
    for impl in ("fused", "torch"):
        eng = engine(impl, hidden_size=hidden, num_attention_heads=heads)
        x, y = batch(0)
        eng.optimizer.zero_grad()
        before = _lib.launch_count()
        loss = eng.forward_loss(x, y)
        loss.backward()
        grads[impl] = {"loss": loss.detach().float(), **{n: p.grad.float().clone() for n, p in eng.model.named_parameters()}}
        if impl == "fused":
            assert _lib.launch_count() - before > 2 * 8
    assert any("q_norm" in n for n in grads["fused"])
    for n, a in grads["fused"].items():
        b = grads["torch"][n]
        assert (a - b).norm() <= 2.0 ** -5 * b.norm(), n


def test_steps_from_a_graph_equal_eager_ones(cuda_device):
    """The mask is made of each step's tokens, in the graph too."""
    losses = []
    for graph in (False, True):
        eng = engine("fused", graph, hidden_size=256, num_attention_heads=4)
        losses.append([float(eng.train_step(*batch(step))) for step in range(7)])
        assert (eng._graph is not None) == graph
        del eng
    assert losses[0] == losses[1]


def test_documents_do_not_see_each_other(cuda_device):
    eng = engine("fused", hidden_size=256, num_attention_heads=4)
    x, _ = batch(3, B=1)
    x[0, 100] = 0
    y = x.clone()
    y[0, 5] = x[0, 5] % 1000 + 1
    with torch.no_grad():
        eng.model.eval()
        a, b = eng.model(x), eng.model(y)
    assert torch.equal(a[101:], b[101:]) and not torch.equal(a[5:101], b[5:101])
