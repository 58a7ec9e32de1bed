"""The model with norms of q and k, capped scores, a window and documents, in fp32 on the CPU."""
import pytest
import torch
import torch.distributed as dist

from dist_utils import run_ranks
from gpt_from_scratch_b200.config import GPTConfig
from gpt_from_scratch_b200.models.gpt import GPTModel
from gpt_from_scratch_b200.ops import RopeScaling
from gpt_from_scratch_b200.parallel import parallel_state as ps

CFG = dict(vocab_size=512, hidden_size=128, num_layers=2, num_attention_heads=4, max_position_embeddings=64,
           intermediate_size=256, init_method="normal", init_std=0.2)


@pytest.fixture
def one_rank():
    ps.set_device("cpu")
    ps.initialize_parallel_state(1)
    ps.set_seed(3)


def tokens(*lengths, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(1, 512, (1, n), generator=g) for n in lengths]


@pytest.mark.parametrize("more", [{}, dict(qk_norm=True, attention_softcap=5.0), dict(attention_window=6)])
def test_packed_documents_are_read_like_separate_ones(one_rank, more):
    model = GPTModel(GPTConfig(**CFG, eod_token_id=0, **more))
    a, b, c = tokens(11, 1, 20)
    end = torch.zeros(1, 1, dtype=torch.long)
    parts = [torch.cat((a, end), 1), torch.cat((b, end), 1), end, c]      # a document may be its end alone
    with torch.no_grad():
        packed = model(torch.cat(parts, 1))
        apart = torch.cat([model(p) for p in parts])
    assert (packed - apart).abs().max() <= 1e-4 * apart.abs().max()


def test_window_and_causality(one_rank):
    model = GPTModel(GPTConfig(**CFG, attention_window=4))
    (x,) = tokens(24)
    y = x.clone()
    y[0, 10] = (x[0, 10] + 1) % 512
    with torch.no_grad():
        moved = (model(x) - model(y)).abs().amax(-1)[:, 0] > 0
    # two blocks of a window of 4 tokens: 3 tokens further each
    assert not moved[:10].any() and moved[10:17].all() and not moved[17:].any()


def test_cap_bounds_what_a_token_can_weigh(one_rank):
    """With a tiny cap all scores are nearly equal: attention becomes the mean, whatever the queries are."""
    model = GPTModel(GPTConfig(**CFG, attention_softcap=1e-4))
    att = model.layers[0].attention
    h = torch.randn(9, 1, 128)
    with torch.no_grad():
        out = att(h, mask=model.attention_mask(torch.ones(1, 9, dtype=torch.long)))
        v = att.qkv_proj(h).view(9, 1, 3, 4, 32)[:, :, 2]
        mean = v.cumsum(0) / torch.arange(1, 10).view(9, 1, 1, 1)
        want = att.out_proj(mean.reshape(9, 1, 128))
    assert (out - want).abs().max() <= 2e-4 * want.abs().max()     # exp(2e-4) - 1


def test_norms_of_q_and_k_get_their_gradients(one_rank):
    """Against differences, in 64 bits: the attention alone, as the block's own norms compute in 32 whatever their input."""
    model = GPTModel(GPTConfig(**CFG, qk_norm=True, eod_token_id=0)).double()
    att = model.layers[1].attention
    x = torch.cat((tokens(9)[0], torch.zeros(1, 1, dtype=torch.long), tokens(8)[0]), 1)
    mask = model.attention_mask(x)
    g = torch.Generator().manual_seed(1)
    h, coef = (torch.randn(18, 1, 128, dtype=torch.float64, generator=g) for _ in range(2))

    def f():
        return (att(h, mask=mask) * coef).sum()
    f().backward()
    for name in ("q_norm", "k_norm"):
        w = getattr(att, name).weight
        d = torch.randn(w.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(2))
        with torch.no_grad():
            w += 1e-5 * d
            up = f()
            w -= 2e-5 * d
            down = f()
            w += 1e-5 * d
        slope, got = float(up - down) / 2e-5, float((w.grad * d).sum())
        assert abs(slope) > 1e-3 and abs(slope - got) <= 1e-5 * max(1.0, abs(slope))


def test_scaled_tables_reach_the_model(one_rank):
    plain, scaled = (GPTModel(GPTConfig(**CFG, rope_scaling=s)) for s in (None, RopeScaling("linear", 2.0)))
    scaled.load_state_dict(plain.state_dict())
    (x,) = tokens(6)
    with torch.no_grad():
        assert (plain(x) - scaled(x)).abs().max() > 1e-3
        cos = scaled.layers[0].attention.rotary_emb.cos_cached
        assert (cos[::2] - plain.layers[0].attention.rotary_emb.cos_cached[:32]).abs().max() < 1e-5


def test_command_line():
    import train
    args = train.parse_args(["--qk-norm", "--attention-softcap", "30", "--attention-window", "512", "--eod-token-id", "50256",
                             "--rope-scaling", "by_parts", "--rope-scaling-factor", "4", "--rope-original-length", "1024"])
    cfg = train.build_config(args)
    assert (cfg.qk_norm, cfg.attention_softcap, cfg.attention_window, cfg.eod_token_id) == (True, 30.0, 512, 50256)
    assert cfg.rope_scaling == RopeScaling("by_parts", 4.0, 1024)
    plain = train.build_config(train.parse_args([]))
    assert plain == GPTConfig(max_position_embeddings=1024) and plain.rope_scaling is None


def _worker(rank, world, tp):
    from gpt_from_scratch_b200.engine import TrainEngine
    from gpt_from_scratch_b200.utils.reshard import merge_state_dicts, shard_state_dict
    ps.set_device("cpu")
    ps.initialize_parallel_state(tp)
    cfg = GPTConfig(**CFG, qk_norm=True, attention_softcap=8.0, eod_token_id=0)
    eng = TrainEngine(cfg, lr=1e-2, dtype=torch.float32, seed=5)
    g = torch.Generator().manual_seed(9)
    full = {}
    for k, v in eng.model.state_dict().items():       # the same weights on every layout, made whole and then cut
        shape = list(v.shape)
        if tp > 1 and k.endswith(("qkv_proj.weight", "gate_up_proj.weight", "embedding.weight", "output.weight")):
            shape[0] *= tp
        elif tp > 1 and k.endswith(("out_proj.weight", "down_proj.weight")):
            shape[1] *= tp
        full[k] = v.clone() if k.endswith("freqs") else torch.randn(shape, generator=g) * (0.1 if v.dim() > 1 else 0.2) + \
            (0.0 if v.dim() > 1 else 1.0)
    eng.model.load_state_dict(shard_state_dict(full, rank, tp))
    eng.optimizer.fp32_master_shard.data.copy_(eng.optimizer.param_buffer[eng.optimizer.shard_start:eng.optimizer.shard_end])
    losses = []
    for step in range(3):
        t = torch.randint(0, 512, (2, 33), generator=torch.Generator().manual_seed(step))
        t[:, 7 + step] = 0
        losses.append(float(eng.train_step(t[:, :-1].contiguous(), t[:, 1:].contiguous())))
    states = [None] * world
    sd = {k: v.clone() for k, v in eng.model.state_dict().items()}
    if world > 1:
        dist.all_gather_object(states, sd)
    else:
        states = [sd]
    return losses, merge_state_dicts(states)


def test_tensor_parallel_ranks_train_the_same_model(tmp_path):
    (whole, one), = run_ranks(_worker, 1, (1,), tmp_path)
    for losses, state in run_ranks(_worker, 2, (2,), tmp_path):
        assert max(abs(a - b) for a, b in zip(whole, losses)) < 1e-4
        # The norms' gradients are sums over all heads, so over the ranks: one that is not summed moves a weight by another of Adam's
        # first steps, which are lr = 1e-2 times a sign. (Elsewhere gradients near zero have signs that rounding decides.)
        for k in (k for k in one if "q_norm" in k or "k_norm" in k):
            assert (one[k] - state[k]).abs().max() < 2e-3, k
