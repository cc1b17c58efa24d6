"""The token mixer of the port block's linear-attention layers, as measurable cases.

Between the mixer's two projections such a layer runs a short causal
convolution over the mixed q, k, v rows, the gated delta rule on its heads and
a gated norm; at the block's edges a norm joins the mixer's output to the
residual stream and normalises it for the MoE section.  Decoding makes each
call with one token per sequence, prompts come as ragged batches of sequences.

Sequences lie back to back in the token rows: sequence i has the rows
offsets[i] .. offsets[i + 1] - 1, its state is slot slots[i] of the state
array, and a sequence marked in `fresh` starts from zeros.  Rows behind the
last sequence and slots without a sequence stay as they are.

A case is a dict of plain values:
  op       "delta"  the gated delta rule on q, k [T][k_heads][k_dim] and
                    v [T][v_heads][v_dim], slices of one mixed row, with raw
                    gates a, b [T][v_heads]; state [slots][v_heads][k_dim][v_dim]
           "conv"   causal depthwise convolution of `width` taps with SiLU,
                    state [slots][width - 1][channels]
           "norm"   u = rmsnorm(x) * gamma (where `post`), times silu or
                    sigmoid of a gate; stream = residual + scale * u; and (where
                    `edge`) y = rmsnorm(stream) * edge_gamma
  type     "bf16", "f16" or "f32": the rows' type
  seqs, tokens, pad   sequences, their tokens in all, rows behind the last one
  rows, groups, dim   norm: rows of `groups` groups of `dim`, each normalised
  stream   norm: the type of the residual stream and of y
"""
import math
import os
import random
import sys

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
CHUNK = 64  # tokens that the plain delta rule takes at once


def _delta(name, seqs, tokens, k_heads=16, v_heads=32, k_dim=128, v_dim=128, type="bf16", pad=0):
    c = {"op": "delta", "type": type, "seqs": seqs, "tokens": tokens, "pad": pad,
         "k_heads": k_heads, "v_heads": v_heads, "k_dim": k_dim, "v_dim": v_dim}
    return dict(c, name=name) if name else c


def _conv(name, seqs, tokens, channels=8192, width=4, bias=False, type="bf16", pad=0):
    c = {"op": "conv", "type": type, "seqs": seqs, "tokens": tokens, "pad": pad,
         "channels": channels, "width": width, "bias": bias}
    return dict(c, name=name) if name else c


def _norm(name, rows, dim, groups=1, type="bf16", stream="f32", post=True, gate="", residual=True,
          vector=False, edge=True):
    c = {"op": "norm", "type": type, "stream": stream, "rows": rows, "groups": groups, "dim": dim,
         "post": post, "gate": gate, "residual": residual, "vector": vector, "edge": edge}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one stream decodes: a layer's 32 heads of one token
        _delta("delta decode 1", 1, 1),
        # some tens of streams decode together
        _delta("delta decode 32", 32, 32),
        # a full serving batch, padded to a captured graph's size
        _delta("delta decode 250 of 256", 250, 250, pad=6),
        # one prompt chunk of the benchmark's prefill length
        _delta("delta prefill 2048", 1, 2048),
        # prompts and single tokens of many requests in one call, a smaller head shape, fp32 rows
        _delta("delta ragged 37 f32", 37, 4711, k_heads=4, v_heads=12, k_dim=64, v_dim=96,
               type="f32"),
        # long prompts of a few requests
        _delta("delta prefill 4 x long", 4, 16384),
        # the convolution of some tens of decoding streams
        _conv("conv decode 32", 32, 32),
        # the convolution of a batch of prompts
        _conv("conv ragged 21", 21, 16384, type="f16", pad=3),
        # the block's edge for one decoded token: residual stream in fp32, as the MoE block takes it
        _norm("edge norm 1 row", 1, 2048, post=False),
        # the same for a batch of prompts, with the norm after the block and a residual scale
        _norm("edge norm 16384 rows", 16384, 2048, vector=True),
        # the delta rule's output norm: 32 heads of a prompt chunk, gated
        _norm("gated head norm 2048", 2048, 128, groups=32, stream="bf16", gate="silu",
              residual=False, edge=False),
        # an odd width, fp32 rows, a sigmoid gate before the residual
        _norm("gated edge norm 517 x 5001", 517, 5001, type="f32", gate="sigmoid"),
    ]


def _log(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    op = rng.choice(["delta", "delta", "delta", "conv", "norm", "norm"])
    type = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "norm":
        groups = rng.choice([1, 1, rng.randint(2, 32)])
        dim = _log(rng, 16, 8192 if groups == 1 else 256)
        edge = rng.random() < 0.6
        return _norm(None, min(_log(rng, 1, 16384), (1 << 25) // (groups * dim)), dim, groups, type,
                     rng.choice([type, "f32"]), post=rng.random() < 0.6 or not edge,
                     gate=rng.choice(["", "silu", "sigmoid"]), residual=rng.random() < 0.7,
                     vector=rng.random() < 0.3, edge=edge)
    seqs = _log(rng, 1, 200)
    tokens = seqs if rng.random() < 0.4 else max(seqs, _log(rng, 16, 8000))
    pad = rng.choice([0, 0, rng.randint(1, 9)])
    if op == "conv":
        return _conv(None, seqs, tokens, _log(rng, 64, 8192), rng.choice([4, 4, 3, 2]),
                     rng.random() < 0.5, type, pad)
    if rng.random() < 0.4:
        heads = {}
    else:
        k_heads = rng.randint(1, 12)
        heads = {"k_heads": k_heads, "v_heads": k_heads * rng.randint(1, 3),
                 "k_dim": 8 * rng.randint(2, 16), "v_dim": 8 * rng.randint(2, 16)}
    return _delta(None, seqs, tokens, type=type, pad=pad, **heads)


# ---- inputs -----------------------------------------------------------------
def _lengths(case):
    """Lengths of a case's sequences: all one where there are as many tokens;
    else skewed ones, an empty sequence and single tokens among them."""
    n, tokens = case["seqs"], case["tokens"]
    if n == tokens:
        return [1] * n
    rng = random.Random(n * 100003 + tokens)
    w = [rng.expovariate(1.0) + 0.05 for _ in range(n)]
    lens = [int(tokens * x / sum(w)) for x in w]
    for i in range(2, n, 5):
        lens[i] = i // 5 % 2
    lens[lens.index(max(lens))] += tokens - sum(lens)
    return lens


def _batch(case, g):
    """Offsets, slots and fresh marks of a case's sequences, with three slots to spare."""
    lens = _lengths(case)
    offsets = [0]
    for n in lens:
        offsets.append(offsets[-1] + n)
    slots = torch.randperm(len(lens) + 3, generator=g, device="cuda")[: len(lens)].int()
    fresh = (torch.rand(len(lens), generator=g, device="cuda") < 0.25).int()
    return {"lens": lens, "offsets": torch.tensor(offsets, dtype=torch.int32, device="cuda"),
            "slots": slots, "fresh": fresh, "num_slots": len(lens) + 3, "max_len": max(lens)}


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    t = TYPES[case["type"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def rand(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    if case["op"] == "norm":
        shape = (case["rows"], case["groups"], case["dim"])
        st = TYPES[case["stream"]]
        # channels of a block's output differ in size
        s = {"x": (randn(*shape) * (0.2 + rand(case["dim"]) * 2)).to(t)}
        s["gamma"] = 1 + 0.2 * randn(case["dim"]) if case["post"] else None
        s["gate"] = randn(*shape).to(t) if case["gate"] else None
        s["residual"] = (2 * randn(*shape)).to(st) if case["residual"] else None
        s["scale"] = 0.1 + rand(case["groups"], case["dim"]) if case["vector"] else 0.7071
        s["edge_gamma"] = 1 + 0.2 * randn(case["dim"]) if case["edge"] else None
        s["stream"] = torch.empty(shape, dtype=st, device="cuda")
        s["y"] = torch.empty(shape, dtype=st, device="cuda") if case["edge"] else None
        return s
    s = _batch(case, g)
    rows = case["tokens"] + case["pad"]
    if case["op"] == "conv":
        c, w = case["channels"], case["width"]
        s["x"] = randn(rows, c).to(t)
        s["weight"] = randn(c, w) * 0.5
        s["bias"] = randn(c) * 0.2 if case["bias"] else None
        s["state"] = randn(s["num_slots"], w - 1, c).to(t)
        s["y"] = torch.full((rows, c), 0.5, dtype=t, device="cuda")
        return s
    hk, hv, dk, dv = (case[k] for k in ("k_heads", "v_heads", "k_dim", "v_dim"))
    # what a convolution with SiLU gives: mostly small values with a positive mean
    x = randn(rows, 2 * hk * dk + hv * dv)
    x = (x * torch.sigmoid(x)).to(t)
    s["q"] = x[:, : hk * dk].unflatten(1, (hk, dk))
    s["k"] = x[:, hk * dk: 2 * hk * dk].unflatten(1, (hk, dk))
    s["v"] = x[:, 2 * hk * dk:].unflatten(1, (hv, dv))
    s["a"], s["b"] = randn(rows, hv).to(t), randn(rows, hv).to(t)
    # decays as such layers are trained from: A in (1, 16), time steps of 0.001 to 0.1
    s["a_log"] = (1 + 15 * rand(hv)).log()
    dt = (rand(hv) * math.log(100) + math.log(0.001)).exp()
    s["dt_bias"] = dt + (-(-dt).expm1()).log()
    s["state"] = randn(s["num_slots"], hv, dk, dv) * 0.1
    s["o"] = torch.full((rows, hv, dv), 2.0 ** -6, dtype=t, device="cuda")
    return s


_blocks = []


def _block():
    """The process's device context."""
    if not _blocks:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                            "disk-streaming-moe-engine_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        from dismoen import MoEBlock
        _blocks.append(MoEBlock(0))
    return _blocks[0]


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        blk = _block()
        from dismoen import GatedDelta, GatedNorm, SeqBatch, ShortConv
        if case["op"] == "norm":
            s["op"] = GatedNorm(blk, case["dim"], case["groups"], gamma=s["gamma"],
                                edge_gamma=s["edge_gamma"], post=case["post"], edge=case["edge"],
                                gate=case["gate"] or None, scale=s["scale"], eps=EPS)
            return s
        s["batch"] = SeqBatch(s["offsets"], case["tokens"], s["max_len"], s["num_slots"],
                              slots=s["slots"], fresh=s["fresh"])
        if case["op"] == "conv":
            s["op"] = ShortConv(blk, s["weight"], bias=s["bias"], silu=True)
        else:
            s["op"] = GatedDelta(blk, case["k_heads"], case["v_heads"], case["k_dim"],
                                 case["v_dim"], a_log=s["a_log"], dt_bias=s["dt_bias"],
                                 qk_norm=True, eps=EPS)
    return s


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "norm":
            s["op"](s["x"], s["stream"], s["y"], gate=s["gate"], residual=s["residual"])
        elif op == "conv":
            s["op"](s["x"], s["state"], s["batch"], s["y"])
        else:
            s["op"](s["q"], s["k"], s["v"], s["a"], s["b"], s["state"], s["batch"], s["o"])
    else:
        {"norm": _plain_norm, "conv": _plain_conv, "delta": _plain_delta}[op](s)
    if op == "norm":
        return {"stream": s["stream"], "y": s["y"]}
    return {"out": s["y" if op == "conv" else "o"], "state": s["state"]}


# ---- the plain forms ----------------------------------------------------------
def _plain_norm(s):
    case = s["case"]
    u = s["x"].float()
    if case["post"]:
        u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS) * s["gamma"]
    if case["gate"]:
        z = s["gate"].float()
        u = u * (z * torch.sigmoid(z) if case["gate"] == "silu" else torch.sigmoid(z))
    r = s["scale"] * u
    if case["residual"]:
        r = s["residual"].float() + r
    s["stream"].copy_(r)
    if case["edge"]:
        s["y"].copy_(r * torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS) * s["edge_gamma"])


def _plain_conv(s):
    case, x, state = s["case"], s["x"], s["state"]
    w, n = case["width"], case["tokens"]
    first, slots = s["offsets"][:-1].long(), s["slots"].long()
    lens = s["offsets"][1:].long() - first
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), lens, output_size=n)
    at = torch.arange(n, device="cuda")
    pos = at - first[seq]
    old = state.float()[slots] * (s["fresh"] == 0)[:, None, None]  # [seqs][w - 1][channels]
    y = 0.0 if s["bias"] is None else s["bias"]
    for back in range(w):  # the taps
        row = torch.where((pos >= back)[:, None], x[(at - back).clamp(min=0)].float(),
                          old[seq, (w - 1 + pos - back).clamp(max=w - 2)])
        y = y + row * s["weight"][:, w - 1 - back]
    s["y"][:n] = (y * torch.sigmoid(y)).to(x.dtype)
    last = lens[:, None] - (w - 1) + torch.arange(w - 1, device="cuda")  # positions kept
    new = torch.where((last >= 0)[:, :, None], x[(first[:, None] + last).clamp(0, n - 1)].float(),
                      old.gather(1, (w - 1 + last).clamp(max=w - 2)[:, :, None].expand_as(old)))
    live = lens > 0
    state[slots[live]] = new[live].to(state.dtype)


def _plain_delta(s):
    case = s["case"]
    hv, rep = case["v_heads"], case["v_heads"] // case["k_heads"]
    first, slots = s["offsets"][:-1].long(), s["slots"].long()
    lens = s["offsets"][1:].long() - first
    size = 1 if s["max_len"] == 1 else CHUNK
    chunks = -(-s["max_len"] // size)
    pos = torch.arange(chunks * size, device="cuda")
    live = pos < lens[:, None]  # [seqs][padded length]
    at = torch.where(live, first[:, None] + pos, 0)

    def heads(x):  # [T][heads][d] -> [seqs][heads][chunks][size][d] in fp32, zeros behind a sequence
        x = torch.where(live[:, :, None, None], x[at].float(), 0.0)
        return x.unflatten(1, (chunks, size)).permute(0, 3, 1, 2, 4)

    def unit(x):
        return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS)

    q = unit(heads(s["q"])).repeat_interleave(rep, 1) * case["k_dim"] ** -0.5
    k = unit(heads(s["k"])).repeat_interleave(rep, 1)
    v = heads(s["v"])
    dt = s["a"].float() + s["dt_bias"]
    step = -s["a_log"].exp() * torch.where(dt > 20, dt, dt.clamp(max=20).exp().log1p())
    beta = heads(torch.sigmoid(s["b"].float())[:, :, None])
    since = heads(step[:, :, None]).double().cumsum(3)  # log decay since the chunk's start
    gone = (since - since.transpose(3, 4)).tril().exp().float().tril()  # from j to i
    low = (beta * (k @ k.transpose(3, 4)) * gone).tril(-1)
    inv = torch.eye(size, device="cuda").expand(low.shape).contiguous()
    for i in range(1, size):  # (I + low)^-1 by forward substitution
        inv[..., i, :] -= (low[..., i, None, :] @ inv).squeeze(-2)
    grow = since.exp().float()
    rest = (since[:, :, :, -1:] - since).exp().float()
    w = inv @ (beta * grow * k)
    u0 = inv @ (beta * v)
    qk = (q @ k.transpose(3, 4)) * gone
    state = torch.where((s["fresh"] == 0)[:, None, None, None], s["state"][slots], 0.0)
    o = torch.empty(len(lens), hv, chunks, size, case["v_dim"], device="cuda")
    for c in range(chunks):
        u = u0[:, :, c] - w[:, :, c] @ state
        o[:, :, c] = grow[:, :, c] * (q[:, :, c] @ state) + qk[:, :, c] @ u
        state = grow[:, :, c, -1:] * state + (rest[:, :, c] * k[:, :, c]).transpose(2, 3) @ u
    o = o.permute(0, 2, 3, 1, 4).flatten(1, 2)
    s["o"][at[live]] = o[live].to(s["o"].dtype)
    some = lens > 0
    s["state"][slots[some]] = state[some]


# ---- in 64 bits, from the definitions -------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "norm":
        u = s["x"].double()
        if case["post"]:
            u = u / (u.square().mean(-1, keepdim=True) + EPS).sqrt() * s["gamma"].double()
        if case["gate"]:
            z = s["gate"].double()
            u = u / (1 + (-z).exp())
            u = u * z if case["gate"] == "silu" else u
        r = u * (s["scale"].double() if case["vector"] else s["scale"])
        if case["residual"]:
            r = r + s["residual"].double()
        y = None
        if case["edge"]:
            y = r / (r.square().mean(-1, keepdim=True) + EPS).sqrt() * s["edge_gamma"].double()
        return {"stream": r, "y": y}
    lens = s["lens"]
    starts = [sum(lens[:i]) for i in range(len(lens))]
    slots = s["slots"].tolist()
    fresh = s["fresh"].tolist()
    state = s["state"].double()
    if case["op"] == "conv":
        x, y, w = s["x"].double(), s["y"].double(), case["width"]
        for n, t, slot, new in zip(lens, starts, slots, fresh):
            if n:
                past = state[slot] * (0.0 if new else 1.0)
                line = torch.cat([past, x[t: t + n]])
                z = (line.unfold(0, w, 1) * s["weight"].double()).sum(-1)
                z = z if s["bias"] is None else z + s["bias"].double()
                y[t: t + n] = z / (1 + (-z).exp())
                state[slot] = line[n:]
        return {"out": y, "state": state}
    # token after token, all sequences that have one left at once
    rep = case["v_heads"] // case["k_heads"]
    o = s["o"].double()
    order = sorted((i for i in range(len(lens)) if lens[i]), key=lambda i: -lens[i])
    sel = torch.tensor([slots[i] for i in order], device="cuda")
    row = torch.tensor([starts[i] for i in order], device="cuda")
    keep = torch.tensor([0.0 if fresh[i] else 1.0 for i in order], device="cuda")
    m = state[sel] * keep.double()[:, None, None, None]
    counts = [lens[i] for i in order]
    a_log, dt_bias = s["a_log"].double(), s["dt_bias"].double()
    left = len(order)
    for t in range(counts[0]):
        while counts[left - 1] <= t:
            left -= 1
        r = row[:left] + t
        q, k = (x[r].double().repeat_interleave(rep, 1) for x in (s["q"], s["k"]))
        q = q / (q.square().sum(-1, keepdim=True) + EPS).sqrt() / math.sqrt(case["k_dim"])
        k = k / (k.square().sum(-1, keepdim=True) + EPS).sqrt()
        g = -a_log.exp() * torch.nn.functional.softplus(s["a"][r].double() + dt_bias)
        beta = torch.sigmoid(s["b"][r].double())
        now = m[:left] * g.exp()[:, :, None, None]
        miss = s["v"][r].double() - (k.unsqueeze(2) @ now).squeeze(2)
        now += k.unsqueeze(3) * (beta.unsqueeze(2) * miss).unsqueeze(2)
        m[:left] = now
        o[r] = (q.unsqueeze(2) @ now).squeeze(2)
    state[sel] = m
    return {"out": o, "state": state}


# ---- what a pass cannot do without ----------------------------------------------
def work(case):
    t = SIZE[case["type"]]
    if case["op"] == "norm":
        n, st = case["rows"] * case["groups"] * case["dim"], SIZE[case["stream"]]
        b = n * t * (2 if case["gate"] else 1) + n * st * (1 + case["residual"] + case["edge"])
        b += 4 * case["dim"] * (case["post"] + case["edge"] + case["groups"] * case["vector"])
        return {"bytes": b, "flops": n * (2 + 4 * case["post"] + 4 * case["edge"]
                                          + 4 * bool(case["gate"]))}
    lens = _lengths(case)
    n, some = case["tokens"], sum(1 for x in lens if x)
    marks = 4 * (3 * case["seqs"] + 1)
    if case["op"] == "conv":
        c, w = case["channels"], case["width"]
        return {"bytes": 2 * n * c * t + 2 * some * (w - 1) * c * t + 4 * c * (w + case["bias"])
                + marks, "flops": n * c * (2 * w + 4)}
    hk, hv, dk, dv = (case[k] for k in ("k_heads", "v_heads", "k_dim", "v_dim"))
    return {"bytes": n * t * (2 * hk * dk + 2 * hv * dv + 2 * hv) + 8 * some * hv * dk * dv
            + 8 * hv + marks, "flops": 6 * n * hv * dk * dv}
