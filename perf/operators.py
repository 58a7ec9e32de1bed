"""Operators of the attention block for packed documents, as cases that can be timed and compared.

Three operators, in their plain form (``own`` false: elementary torch operations, in 32 bits, rounded once at
the end) or as a user of the framework calls them (``own`` true):

* ``rotary``: the position rotation of a ``[S, B, heads, D]`` tensor, pairs side by side or half a head apart,
  of the whole head or of its first dimensions, at positions that are given for every token;
* ``norm_rope``: the packed projection ``[S, B, (heads + 2 kv_heads) * D]`` -> q and k, normalised per head
  (RMS over D, one weight for q and one for k), then rotated;
* ``attend``: attention under a mask made of documents, a prefix (prompt) that all of its document sees, a
  window and padding; scores capped by a tanh, or with a bias that falls with the distance.

``train`` cases run the backward pass too and return the gradients. A case is a dict of plain values. The
lengths of a case's documents are the same for every seed, their order is not, so a case has one amount of work.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _rotary(name, seq, batch, heads, head_dim, rotary_dim, interleaved, dtype="bf16", documents=0, packed=False,
            train=False, far=0):
    return dict(name=name, op="rotary", seq=seq, batch=batch, heads=heads, head_dim=head_dim, rotary_dim=rotary_dim,
                interleaved=interleaved, dtype=dtype, documents=documents, packed=packed, train=train, far=far)


def _norm_rope(name, seq, batch, heads, kv_heads, head_dim, interleaved=True, dtype="bf16", documents=0, train=False):
    return dict(name=name, op="norm_rope", seq=seq, batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                rotary_dim=head_dim, interleaved=interleaved, dtype=dtype, documents=documents, train=train, far=0)


def _attend(name, seq, batch, heads, kv_heads, head_dim, documents=0, padding=0, prefix=0.0, window=0, cap=0.0,
            distance=False, train=True):
    return dict(name=name, op="attend", seq=seq, batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                dtype="bf16", documents=documents, padding=padding, prefix=prefix, window=window, cap=cap,
                distance=distance, train=train)


def listed():
    return [
        # One token for each of eight sequences, far into a long context: the smallest call, all latency.
        _rotary("rotary-one-token", 1, 8, 12, 64, 64, True, far=100000),
        # A ragged micro-batch in 32 bits, the type that the framework trains in on a CPU and checks itself with.
        _rotary("rotary-ragged-fp32", 777, 3, 12, 64, 64, True, dtype="fp32", documents=100, train=True),
        # Half the head rotated, halves apart, read out of the packed projection of the 1.3B model: a training step.
        _rotary("rotary-partial-train", 2048, 4, 16, 128, 64, False, documents=300, packed=True, train=True),
        # A short text scored by the default model: again latency.
        _norm_rope("norm-rope-short", 130, 1, 12, 12, 64),
        # The default model's micro-batch of the benchmark, its sequences packed with documents.
        _norm_rope("norm-rope-124m-train", 1024, 16, 12, 12, 64, documents=200, train=True),
        # The 7B shape with shared key heads, fp16, halves apart: the largest of its kind.
        _norm_rope("norm-rope-grouped-train", 4096, 2, 32, 8, 128, interleaved=False, dtype="fp16", documents=500,
                   train=True),
        # A single token: the shortest sequence there is.
        _attend("attend-one-token", 1, 8, 12, 12, 64, train=False),
        # The default model's micro-batch of the benchmark, packed with documents of 200 tokens on average.
        _attend("attend-documents-train", 1024, 16, 12, 12, 64, documents=200),
        # A distance bias in place of rotated positions, an odd length, padding behind the last document.
        _attend("attend-distance-ragged-train", 777, 3, 12, 12, 64, documents=300, padding=77, distance=True),
        # Capped scores, shared key heads, the sequence length of the 1.3B model.
        _attend("attend-capped-train", 2048, 4, 16, 4, 128, documents=600, cap=30.0),
        # A local layer of the 7B shape scoring a long text: window and cap, forward only.
        _attend("attend-window-capped", 4096, 2, 32, 8, 128, window=1024, cap=50.0, train=False),
        # Prompts and answers packed into a long context; every token of a document sees its whole prompt.
        _attend("attend-prefix-long-train", 8192, 1, 16, 4, 128, documents=3000, prefix=0.3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "norm_rope", "attend", "attend"])
    train = rng.random() < 0.6
    if op == "attend":
        head_dim = rng.choice([64, 128])
        kv = rng.choice([1, 2, 3, 4, 8, 12])
        heads = kv * rng.choice([1, 1, 2, 4])
        seq = min(_log(rng, 2 if not train else 16, 6000), math.isqrt(900_000_000 // heads))
        batch = max(1, min(_log(rng, 1, 16), 600_000_000 // (seq * seq * heads)))
        return dict(op=op, seq=seq, batch=batch, heads=heads, kv_heads=kv, head_dim=head_dim, dtype="bf16",
                    documents=rng.choice([0, max(4, seq // 2), max(4, seq // 5)]),
                    padding=rng.choice([0, 0, seq // 10]), prefix=rng.choice([0.0, 0.0, 0.4]),
                    window=rng.choice([0, 0, max(1, seq // 3)]), cap=rng.choice([0.0, 15.0, 50.0]),
                    distance=rng.random() < 0.3, train=train)
    seq, batch = _log(rng, 1, 6000), _log(rng, 1, 16)
    kv = rng.choice([1, 2, 4, 8, 12])
    heads = kv * rng.choice([1, 2, 4])
    head_dim = rng.choice([64, 80, 96, 128, 256])
    batch = max(1, min(batch, 67_000_000 // (seq * (heads + 2 * kv) * head_dim)))
    case = dict(op=op, seq=seq, batch=batch, heads=heads, head_dim=head_dim, interleaved=rng.random() < 0.5,
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), documents=rng.choice([0, max(4, seq // 3)]),
                train=train, far=0)
    if op == "rotary":
        return dict(case, rotary_dim=rng.choice([head_dim, head_dim // 2, head_dim // 4]), packed=rng.random() < 0.5,
                    far=rng.choice([0, 30000]))
    return dict(case, kv_heads=kv, rotary_dim=head_dim)


# ---------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """The lengths of a row's documents (log-normal around ``documents`` tokens), padding apart."""
    left = case["seq"] - case.get("padding", 0)
    if not case["documents"]:
        return [left]
    rng = random.Random(case["seq"] * 1009 + case["documents"])
    lengths = []
    while left > 0:
        n = min(left, max(1, int(case["documents"] * rng.lognormvariate(-0.3, 0.8))))
        lengths.append(n)
        left -= n
    return lengths


def _prefix_len(case, n):
    return min(n, int(n * case["prefix"]))


def _documents(case, seed):
    """(document of every token, -1 for padding; place of every token in its document; prefix tokens), [B, S]."""
    rng = random.Random(seed)
    ids, places, prefixes = [], [], []
    for _ in range(case["batch"]):
        lengths = _lengths(case)
        rng.shuffle(lengths)
        a, b, c = [], [], []
        for i, n in enumerate(lengths):
            a += [i] * n
            b += range(n)
            c += [j < _prefix_len(case, n) for j in range(n)] if case.get("prefix") else [False] * n
        pad = case["seq"] - len(a)
        ids.append(a + [-1] * pad)
        places.append(b + list(range(pad)))
        prefixes.append(c + [False] * pad)
    to = dict(device="cuda")
    return (torch.tensor(ids, dtype=torch.int32, **to), torch.tensor(places, dtype=torch.int32, **to),
            torch.tensor(prefixes, dtype=torch.bool, **to))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    S, B, nh, D = case["seq"], case["batch"], case["heads"], case["head_dim"]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * std).to(dtype)

    ids, places, prefixes = _documents(case, seed)
    state = dict(case=case)
    if case["op"] == "attend":
        nkv = case["kv_heads"]
        # q, k and v lie in the packed projection [S, B, heads, D], as the model has them; queries are
        # larger than keys, so that some rows attend to few keys
        qkv = normal(S, B, nh + 2 * nkv, D)
        qkv[:, :, :nh] *= 2.0
        state["q"], state["k"], state["v"] = (t.permute(1, 2, 0, 3) for t in qkv.split([nh, nkv, nkv], dim=2))
        state["dout"] = normal(S, B, nh, D).permute(1, 2, 0, 3)
        state["ids"] = ids if case["documents"] or case["padding"] else None
        state["prefixes"] = prefixes if case["prefix"] else None
        state["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / nh) for h in range(nh)], device="cuda") \
            if case["distance"] else None
        return state
    # positions start at zero in every document; those of single tokens lie far into a long context
    R = case["rotary_dim"]
    state["positions"] = None
    first = torch.zeros(B, 1, dtype=torch.int32, device="cuda")
    if case["far"]:
        first = torch.randint(case["far"] // 2, case["far"], (B, 1), device="cuda", generator=gen, dtype=torch.int32)
    if case["documents"] or case["far"]:
        state["positions"] = places + first
    n = S + case["far"]
    angles = torch.outer(torch.arange(n, dtype=torch.float64, device="cuda"),
                         10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R))
    state["cos"], state["sin"] = angles.cos().float(), angles.sin().float()
    if case["op"] == "rotary":
        # as one part of a packed [S, B, 3, heads, D] projection, or alone
        state["x"] = normal(S, B, 3, nh, D)[:, :, 1] if case["packed"] else normal(S, B, nh, D)
        state["dout"] = normal(S, B, nh, D)
        return state
    nkv = case["kv_heads"]
    state["qkv"] = normal(S, B, (nh + 2 * nkv) * D, std=1.7)
    state["wq"], state["wk"] = ((1.0 + 0.2 * torch.randn(D, device="cuda", generator=gen)).to(dtype) for _ in range(2))
    state["dq"], state["dk"], state["dv"] = normal(S, B, nh, D), normal(S, B, nkv, D), normal(S, B, nkv, D)
    return state


# ---------------------------------------------------------------------------------------------- plain forms
def _angles(s, S):
    """cos and sin of every token, [S, B or 1, 1, R / 2]."""
    if s["positions"] is None:
        return s["cos"][:S, None, None], s["sin"][:S, None, None]
    at = s["positions"].t().long()
    return s["cos"][at][:, :, None], s["sin"][at][:, :, None]


def _rotate(x, cos, sin, R, interleaved):
    """The first R dimensions of x [S, B, heads, D] (fp32) rotated by pairs."""
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return y if R == x.shape[-1] else torch.cat((y, x[..., R:]), dim=-1)


def _plain_rotary(s):
    case, x = s["case"], s["x"]
    cos, sin = _angles(s, case["seq"])
    out = _rotate(x.float(), cos, sin, case["rotary_dim"], case["interleaved"]).to(x.dtype)
    if not case["train"]:
        return [out]
    dx = _rotate(s["dout"].float(), cos, -sin, case["rotary_dim"], case["interleaved"]).to(x.dtype)
    return [out, dx]


EPS = 1e-5


def _plain_norm_rope(s):
    case, qkv = s["case"], s["qkv"]
    S, B, nh, nkv, D, R = (case[n] for n in ("seq", "batch", "heads", "kv_heads", "head_dim", "rotary_dim"))
    cos, sin = _angles(s, S)
    x = qkv.float().view(S, B, nh + 2 * nkv, D)[:, :, :nh + nkv]
    w = torch.cat((s["wq"].float().expand(nh, D), s["wk"].float().expand(nkv, D)))
    rstd = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    n = x * rstd
    y = _rotate(n * w, cos, sin, R, case["interleaved"]).to(qkv.dtype)
    q, k = y[:, :, :nh], y[:, :, nh:]
    if not case["train"]:
        return [q, k]
    dy = torch.cat((s["dq"], s["dk"]), dim=2).float()
    dz = _rotate(dy, cos, -sin, R, case["interleaved"])
    dw = (dz * n).sum((0, 1))
    dn = dz * w
    dx = rstd * (dn - n * (dn * n).mean(-1, keepdim=True))
    dqkv = torch.cat((dx.to(qkv.dtype), s["dv"]), dim=2).view_as(qkv)
    return [q, k, dqkv, dw[:nh].sum(0).to(qkv.dtype), dw[nh:].sum(0).to(qkv.dtype)]


def _visible(s):
    """[B, S, S], query by key: what the mask leaves."""
    case = s["case"]
    S = case["seq"]
    i = torch.arange(S, device="cuda")[:, None]
    j = torch.arange(S, device="cuda")[None, :]
    ids = s["ids"] if s["ids"] is not None else torch.zeros(case["batch"], S, dtype=torch.int32, device="cuda")
    see = (j <= i)[None]
    if s["prefixes"] is not None:
        see = see | s["prefixes"][:, None, :]       # the prefix is the head of the document in these cases
    see = see & (ids[:, :, None] == ids[:, None, :]) & (ids >= 0)[:, :, None]
    if case["window"]:
        see = see & (j > i - case["window"])
    return see


def _plain_attend(s):
    case = s["case"]
    S, B, nh, nkv, D = (case[n] for n in ("seq", "batch", "heads", "kv_heads", "head_dim"))
    group, scale, cap = nh // nkv, 1.0 / math.sqrt(D), case["cap"]
    q = s["q"].float().unflatten(1, (nkv, group))                  # [B, nkv, group, S, D]
    k, v = (s[n].float().unsqueeze(2) for n in ("k", "v"))         # [B, nkv, 1, S, D]
    see = _visible(s)[:, None, None]
    t = torch.matmul(q, k.transpose(-1, -2)) * scale
    if cap:
        t = torch.tanh(t / cap)
    y = t * cap if cap else t
    if case["distance"]:
        i = torch.arange(S, device="cuda")
        y = y - s["slopes"].view(nkv, group, 1, 1) * (i[:, None] - i).abs()
    y = y.masked_fill(~see, float("-inf"))
    top = y.amax(-1, keepdim=True).clamp_min(-3.0e38)
    p = torch.exp(y - top)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    out = torch.matmul(p, v)
    result = [out.flatten(1, 2).to(torch.bfloat16)]
    if not case["train"]:
        return result
    do = s["dout"].float().unflatten(1, (nkv, group))
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
    dy = p * (torch.matmul(do, v.transpose(-1, -2)) - (do * out).sum(-1, keepdim=True))
    if cap:
        dy = dy * (1.0 - t * t)
    dq = torch.matmul(dy, k) * scale
    dk = torch.matmul(dy.transpose(-1, -2), q).sum(2) * scale
    return result + [dq.flatten(1, 2).to(torch.bfloat16), dk.to(torch.bfloat16), dv.to(torch.bfloat16)]


# ---------------------------------------------------------------------------------------------- the framework's calls
def _own_rotary(s):
    from gpt_from_scratch_b200 import ops
    case, x = s["case"], s["x"].detach()
    x.requires_grad_(case["train"])
    out = ops.rotary(x, s["cos"], s["sin"], positions=s["positions"], interleaved=case["interleaved"])
    if not case["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, x, s["dout"])]


def _own_norm_rope(s):
    from gpt_from_scratch_b200 import ops
    case = s["case"]
    leaves = [s[n].detach().requires_grad_(case["train"]) for n in ("qkv", "wq", "wk")]
    q, k, v = ops.qk_norm_rope(*leaves, s["cos"], s["sin"], case["heads"], case["kv_heads"], eps=EPS,
                               positions=s["positions"], interleaved=case["interleaved"])
    if not case["train"]:
        return [q, k]
    return [q.detach(), k.detach(), *torch.autograd.grad((q, k, v), leaves, (s["dq"], s["dk"], s["dv"]))]


def _own_attend(s):
    from gpt_from_scratch_b200 import ops
    case = s["case"]
    q, k, v = (s[n].detach().requires_grad_(case["train"]) for n in ("q", "k", "v"))
    mask = ops.attention_mask(case["batch"], case["seq"], document_ids=s["ids"], prefix_mask=s["prefixes"],
                              window=case["window"] or None, device=q.device)
    out = ops.masked_attention(q, k, v, mask, softcap=case["cap"], alibi_slopes=s["slopes"])
    if not case["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, (q, k, v), s["dout"])]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "norm_rope": _own_norm_rope, "attend": _own_attend}[op](state)
    return {"rotary": _plain_rotary, "norm_rope": _plain_norm_rope, "attend": _plain_attend}[op](state)


# ---------------------------------------------------------------------------------------------- work and exact values
def _pairs(case):
    """Pairs of a query and a key that it sees, in one row of the batch."""
    total, w = 0, case["window"]
    for n in _lengths(case):
        p = _prefix_len(case, n)
        if not w:
            total += n * (n + 1) // 2 + p * (p - 1) // 2
        else:
            # token i of the document sees [max(0, i - w + 1), max(i + 1, p))
            total += sum(max(i + 1, p) - max(0, i - w + 1) for i in range(n))
    return total


def work(case):
    S, B, nh, D = (case[n] for n in ("seq", "batch", "heads", "head_dim"))
    size = 4 if case["dtype"] == "fp32" else 2
    tokens = S * B
    if case["op"] == "attend":
        rows = tokens * D * size
        nkv = case["kv_heads"]
        fwd = rows * (2 * nh + 2 * nkv)                            # q, k, v and the output
        bwd = rows * (2 * nh + 2 * nkv) if case["train"] else 0    # dout, dq, dk, dv
        products = 6 if case["train"] else 2                       # Q K', P V; dO V', P' dO, dS K, dS' Q
        return {"bytes": fwd + bwd, "flops": 2 * D * products * _pairs(case) * B * nh}
    R = case["rotary_dim"]
    tables = 4 * R * min(S, tokens)
    if case["op"] == "rotary":
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * tokens * nh * D * size) + tables, "flops": passes * 3 * R * tokens * nh}
    nkv = case["kv_heads"]
    qk, v = tokens * (nh + nkv) * D, tokens * nkv * D
    if not case["train"]:
        return {"bytes": 2 * qk * size + tables, "flops": 7 * qk}
    return {"bytes": (2 * qk + 2 * (qk + v)) * size + tables, "flops": 20 * qk}


def exact(case, seed):
    s = prepare(case, seed)
    S, B, nh, D = (case[n] for n in ("seq", "batch", "heads", "head_dim"))
    f64 = torch.float64
    if case["op"] == "attend":
        return _exact_attend(case, s)
    # every pair as a complex number, turned by its angle
    if s["positions"] is None:
        at = torch.arange(S, device="cuda")[:, None].expand(S, B)
    else:
        at = s["positions"].t().long()
    turn = torch.complex(s["cos"].to(f64), s["sin"].to(f64))[at].unsqueeze(2)
    R = case["rotary_dim"]

    def rotate(x):
        head, tail = x[..., :R], x[..., R:]
        if case["interleaved"]:
            z = torch.view_as_complex(head.unflatten(-1, (R // 2, 2)).contiguous()) * turn
            head = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.view_as_complex(head.unflatten(-1, (2, R // 2)).transpose(-1, -2).contiguous()) * turn
            head = torch.view_as_real(z).transpose(-1, -2).flatten(-2)
        return torch.cat((head, tail), dim=-1)

    if case["op"] == "rotary":
        x = s["x"].to(f64).requires_grad_()
        out = rotate(x)
        if not case["train"]:
            return [out.detach()]
        return [out.detach(), *torch.autograd.grad(out, x, s["dout"].to(f64))]
    nkv = case["kv_heads"]
    qkv, wq, wk = (s[n].to(f64).requires_grad_() for n in ("qkv", "wq", "wk"))
    q, k, v = qkv.view(S, B, nh + 2 * nkv, D).split([nh, nkv, nkv], dim=2)
    q = rotate(q / (q.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * wq)
    k = rotate(k / (k.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * wk)
    if not case["train"]:
        return [q.detach(), k.detach()]
    grads = torch.autograd.grad((q, k, v), (qkv, wq, wk), [s[n].to(f64) for n in ("dq", "dk", "dv")])
    return [q.detach(), k.detach(), *grads]


def _exact_attend(case, s):
    """Head by head, from each query's first and last key, the gradients by differentiation."""
    S, B, nh, nkv, D = (case[n] for n in ("seq", "batch", "heads", "kv_heads", "head_dim"))
    f64 = torch.float64
    out = torch.zeros(B, nh, S, D, dtype=f64, device="cuda")
    grads = [torch.zeros(B, n, S, D, dtype=f64, device="cuda") for n in (nh, nkv, nkv)]
    at = torch.arange(S, device="cuda")
    for b in range(B):
        ids = s["ids"][b].tolist() if s["ids"] is not None else [0] * S
        prefixes = s["prefixes"][b].tolist() if s["prefixes"] is not None else [False] * S
        first, last = [0] * S, [0] * S                             # keys [first, last) of every query
        start = reach = 0
        for i in range(S):
            if i == 0 or ids[i] != ids[i - 1]:
                start = reach = i
                while reach < S and prefixes[reach] and ids[reach] == ids[i]:
                    reach += 1
            first[i] = max(start, i - case["window"] + 1) if case["window"] else start
            last[i] = max(i + 1, reach) if ids[i] >= 0 else first[i]
        first, last = (torch.tensor(t, device="cuda")[:, None] for t in (first, last))
        hidden = (at < first) | (at >= last)
        empty = first >= last
        for h in range(nh):
            g = h * nkv // nh
            q, k, v = (t.to(f64).requires_grad_() for t in (s["q"][b, h], s["k"][b, g], s["v"][b, g]))
            score = q @ k.t() / math.sqrt(D)
            if case["cap"]:
                score = case["cap"] * torch.tanh(score / case["cap"])
            if case["distance"]:
                score = score - s["slopes"][h].to(f64) * (at[:, None] - at).abs()
            # a query without keys answers zeros: its scores are taken out before the softmax
            weight = torch.softmax(score.masked_fill(hidden & ~empty, -math.inf), dim=-1)
            o = weight.masked_fill(empty, 0.0) @ v
            out[b, h] = o.detach()
            if case["train"]:
                for total, n, part in zip(grads, (h, g, g), torch.autograd.grad(o, (q, k, v), s["dout"][b, h].to(f64))):
                    total[b, n] += part
    return [out, *grads] if case["train"] else [out]
