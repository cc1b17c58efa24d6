"""The full-attention layers' operators and the 4-bit projections, as measurable cases.

A full-attention layer's mixer keeps its keys and values in 4 bits: rows are
quantised as they are written to a paged cache, and attention reads the codes.
The projections around both kinds of mixer have 4-bit weights with group scales.

The cache holds blocks of 32 elements of a head's row as 4-bit codes of
+-{0, 0.5, 1, 1.5, 2, 3, 4, 6} with one power of two, the smallest that leaves no
element above 7 (elements above 6 become 6; nearest value, ties to the even code).
Sequences lie back to back in the token rows, sequence i has the rows
offsets[i] .. offsets[i + 1] - 1 and slot slots[i]; its rows' positions follow the
past[slot] tokens that the cache held before, whose pages are pages[slot].  Rows
behind the last sequence stay as they are.

A case is a dict of plain values:
  op       "store"   k, v [T][kv_heads][dim], slices of one projected row, go into
                     the cache and are read back as the values that it holds
           "attend"  q [T][heads][dim] over each sequence's past and its own rows
                     up to itself; where `gate`, times sigmoid of a gate that lies
                     beside q
           "linear"  y = W x (+ bias) with 4-bit W [n][k] in groups along k, each
                     weight scale * code rounded to bf16, as the dequantiser gives it
  type     "bf16", "f16" or "f32": the rows' type; out: linear's result type
  seqs, tokens, pad, past   sequences, their rows in all, rows behind the last one,
                            and the tokens in all that the cache held before
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def _store(name, seqs, tokens, past, kv_heads=2, dim=256, page=64, type="bf16", pad=0):
    c = {"op": "store", "type": type, "seqs": seqs, "tokens": tokens, "past": past, "pad": pad,
         "kv_heads": kv_heads, "dim": dim, "page": page}
    return dict(c, name=name) if name else c


def _attend(name, seqs, tokens, past, heads=16, kv_heads=2, dim=256, page=64, type="bf16",
            gate=True, pad=0):
    c = {"op": "attend", "type": type, "seqs": seqs, "tokens": tokens, "past": past, "pad": pad,
         "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "gate": gate}
    return dict(c, name=name) if name else c


def _linear(name, rows, n, k, group=32, type="bf16", out="bf16", bias=False):
    c = {"op": "linear", "type": type, "out": out, "rows": rows, "n": n, "k": k, "group": group,
         "bias": bias}
    return dict(c, name=name) if name else c


def listed():
    return [
        # a decoding step's new rows of some tens of streams
        _store("store decode 32", 32, 32, 60000),
        # a batch of prompts, some of them continued
        _store("store prompts", 21, 16384, 9000, kv_heads=8, dim=128, type="f16", pad=3),
        # one stream decodes behind a short conversation
        _attend("attend decode 1", 1, 1, 1087, page=16),
        # a serving batch decodes, contexts of all lengths, padded to a captured graph's size
        _attend("attend decode 61 of 64", 61, 61, 262144, pad=3),
        # one stream at the end of a very long document
        _attend("attend decode 1 long", 1, 1, 131071, heads=32, kv_heads=8, dim=128, page=256,
                type="f16", gate=False),
        # a head per key head, fp32 rows
        _attend("attend decode 24 f32", 24, 24, 50000, heads=12, kv_heads=12, dim=64, page=32,
                type="f32", gate=False),
        # one prompt chunk of the benchmark's prefill length
        _attend("attend prefill 2048", 1, 2048, 0),
        # prompts, continued prompts and single tokens of many requests in one call
        _attend("attend ragged 19", 19, 6001, 40000, heads=32, kv_heads=8, dim=128, page=16,
                type="f16", gate=False, pad=5),
        # one token through the queries', gates', keys' and values' projection
        _linear("linear 1 row", 1, 9216, 2048),
        # the output projection of some tens of streams, for the fp32 residual stream
        _linear("linear 32 rows", 32, 2048, 4096, out="f32"),
        # a few positions through a vocabulary's head, an odd number of tokens in it
        _linear("linear 5 rows head", 5, 100003, 2048, group=128, type="f16", out="f32"),
        # the first projection of a prompt chunk
        _linear("linear 2048 rows", 2048, 9216, 2048, bias=True),
    ]


def _log(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "linear", "linear", "store"])
    type = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "linear":
        k = 32 * _log(rng, 4, 200)
        group = rng.choice([g for g in (32, 64, 128, 256) if k % g == 0])
        n = _log(rng, 16, 16384)
        rows = max(1, min(_log(rng, 1, 2048), (1 << 35) // (n * k)))
        return _linear(None, rows, n, k, group, type, rng.choice([type, "f32"]),
                       rng.random() < 0.3)
    dim = rng.choice([32, 64, 96, 128, 128, 192, 256])
    kv_heads = rng.randint(1, 8)
    page = rng.choice([16, 32, 64, 128, 256])
    pad = rng.choice([0, 0, rng.randint(1, 9)])
    seqs = _log(rng, 1, 100)
    if op == "store":
        tokens = seqs if rng.random() < 0.5 else max(seqs, _log(rng, 16, 16000))
        return _store(None, seqs, tokens, _log(rng, 1, 20000), kv_heads, dim, page, type, pad)
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 6, 8, 16])
    gate = rng.random() < 0.5
    if rng.random() < 0.6:  # single tokens
        past = min(_log(rng, 64, 260000), (1 << 28) // (kv_heads * dim))
        return _attend(None, seqs, seqs, past, heads, kv_heads, dim, page, type, gate, pad)
    seqs = min(seqs, 20)
    tokens = min(max(2 * seqs, _log(rng, 32, 6000)), (1 << 23) // (heads * dim))
    tokens = max(tokens, 2 * seqs)
    past = min(_log(rng, 64, 40000), (1 << 28) // (kv_heads * dim))
    # no more scores than the largest listed cases have
    while tokens * (past + tokens) * heads * dim > 1 << 38 and past > 64:
        past //= 2
    return _attend(None, seqs, tokens, past, heads, kv_heads, dim, page, type, gate, pad)


# ---- inputs -----------------------------------------------------------------
def _shares(n, total, rng, least=0):
    """n skewed whole numbers of sum `total`."""
    w = [rng.expovariate(1.0) + 0.05 for _ in range(n)]
    left = total - least * n
    parts = [least + int(left * x / sum(w)) for x in w]
    parts[parts.index(max(parts))] += total - sum(parts)
    return parts


def _lengths(case):
    """(rows, tokens before) of each sequence: all rows one where there are as many
    sequences, else skewed, single ones among them; some sequences begin."""
    n, tokens = case["seqs"], case["tokens"]
    rng = random.Random(n * 100003 + tokens * 7 + case["past"])
    if n == tokens:
        rows = [1] * n
    else:
        rows = _shares(n, tokens, rng, 1)
        for i in range(2, n, 4):
            rows[rows.index(max(rows))] += rows[i] - 1
            rows[i] = 1
    past = _shares(n, case["past"], rng)
    if n > 4 and n != tokens:
        for i in range(1, n, 3):
            past[past.index(max(past))] += past[i]
            past[i] = 0
    return rows, past


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 29)
    t = TYPES[case["type"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if case["op"] == "linear":
        n, k = case["n"], case["k"]
        q = torch.randint(-7, 8, (n * k,), generator=g, device="cuda", dtype=torch.int8)
        packed = ((q[0::2] & 15) | ((q[1::2] & 15) << 4)).view(torch.uint8)
        scales = (randn(n * k // case["group"]).abs() * 0.02 / 7.5 + 1e-4).half()
        return {"q": q.view(n, k) if not own else None, "packed": packed, "scales": scales,
                "bias": randn(n) * 0.1 if case["bias"] else None, "x": randn(case["rows"], k).to(t)}
    rows, past = _lengths(case)
    h, d, page = case["kv_heads"], case["dim"], case["page"]
    offsets = [0]
    for r in rows:
        offsets.append(offsets[-1] + r)
    n, slots_n = len(rows), len(rows) + 2
    slots = torch.randperm(slots_n, generator=g, device="cuda")[:n]
    need = [-(-(a + b) // page) for a, b in zip(rows, past)]
    ids = torch.randperm(sum(need) + 3, generator=g, device="cuda").int()
    pages = torch.full((slots_n, max(need)), -1, dtype=torch.int32, device="cuda")
    before = torch.zeros(slots_n, dtype=torch.int32, device="cuda")
    where, at = slots.tolist(), 0
    for slot, b, p in zip(where, past, need):
        pages[slot, :p] = ids[at:at + p]
        before[slot] = b
        at += p
    s = {"rows": rows, "past": past, "slots_list": where, "pages": pages, "before": before,
         "num_pages": sum(need) + 3, "num_slots": slots_n, "slots": slots.int(),
         "offsets": torch.tensor(offsets, dtype=torch.int32, device="cuda")}
    total = case["tokens"] + case["pad"]
    size = 0.3 + torch.rand(2, h, d, generator=g, device="cuda") * 1.4  # channels differ in size
    if case["op"] == "store":
        x = (randn(total, 2, h, d) * size).to(t)
        s["k"], s["v"] = x[:, 0], x[:, 1]
        s["k_out"], s["v_out"] = (torch.full((total, h, d), 0.25, dtype=t, device="cuda")
                                  for _ in range(2))
        return s
    # everything that the cache is to hold: each sequence's past and its own rows
    s["context"] = [(randn(2, a + b, h, d) * size[:, None]).to(t) for a, b in zip(rows, past)]
    x = (randn(total, case["heads"], 2, d) * 1.5).to(t)
    s["q"] = x[:, :, 0]
    s["gate"] = x[:, :, 1] if case["gate"] else None
    s["o"] = torch.full((total, case["heads"], d), 0.25, dtype=t, device="cuda")
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
    if case["op"] == "linear":
        if own:
            blk = _block()
            from dismoen import QuantLinear
            torch.cuda.synchronize()
            s["op"] = QuantLinear(blk, case["n"], case["k"], s.pop("scales"),
                                  s.pop("packed"), group_size=case["group"], bias=s["bias"])
            s["y"] = torch.empty(case["rows"], case["n"], dtype=TYPES[case["out"]], device="cuda")
        return s
    h, d, page = case["kv_heads"], case["dim"], case["page"]
    s["codes"] = torch.zeros(s["num_pages"], 2, h, page, d // 2, dtype=torch.uint8, device="cuda")
    s["scales"] = torch.zeros(s["num_pages"], 2, h, page, d // 32, dtype=torch.uint8,
                              device="cuda")
    if own:
        blk = _block()
        from dismoen import CacheAttention, KVCache, SeqBatch
        s["cache"] = KVCache(blk, s["codes"], s["scales"], s["pages"], s["before"])
        s["batch"] = SeqBatch(s["offsets"], case["tokens"], max(s["rows"]), s["num_slots"],
                              slots=s["slots"])
        if case["op"] == "attend":
            s["op"] = CacheAttention(blk, case["heads"])
    if case["op"] == "attend":
        context = s.pop("context")
        if own:
            for i, c in enumerate(context):
                n = c.shape[1]
                whole = SeqBatch(torch.tensor([0, n], dtype=torch.int32, device="cuda"), n, n,
                                 s["num_slots"], slots=s["slots"][i:i + 1],
                                 fresh=torch.ones(1, dtype=torch.int32, device="cuda"))
                torch.cuda.synchronize()
                s["cache"].write(c[0], c[1], whole)
                blk.sync()
        else:
            for i, c in enumerate(context):
                places = _plain_places(s, s["slots_list"][i],
                                       torch.arange(c.shape[1], device="cuda"))
                _plain_write(s, places, c[0], c[1])
    return s


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        if op == "linear":
            return s["op"](s["x"], s["y"])
        if op == "store":
            s["cache"].write(s["k"], s["v"], s["batch"])
            s["cache"].read(s["k_out"], s["v_out"], s["batch"])
            return {"k": s["k_out"], "v": s["v_out"]}
        return s["op"](s["q"], s["cache"], s["batch"], s["o"], gate=s["gate"])
    return {"linear": _plain_linear, "store": _plain_store, "attend": _plain_attend}[op](s)


# ---- the plain forms ----------------------------------------------------------
def _plain_quantise(x):
    """(codes, scale bytes) of rows [..., dim]."""
    x = x.float().unflatten(-1, (-1, 32))
    most = x.abs().amax(-1)
    m, e = torch.frexp(most)  # most = m 2^e, m in [1/2, 1)
    power = torch.where(most > 0, e - 3 + (m > 0.875), -120).clamp(-120, 125)
    y = torch.ldexp(x, -power.unsqueeze(-1)).abs()
    code = ((y > 0.25).int() + (y >= 0.75).int() + (y > 1.25).int() + (y >= 1.75).int()
            + (y > 2.5).int() + (y >= 3.5).int() + (y > 5).int())
    code = (code + 8 * (x < 0).int()).to(torch.uint8).flatten(-2)
    return code, (power + 127).to(torch.uint8)


def _plain_values(codes, scales):
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6],
                         device="cuda")
    x = table[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()]
    return torch.ldexp(x.unflatten(-1, (-1, 32)), scales.int().unsqueeze(-1) - 127).flatten(-2)


def _plain_places(s, slot, pos):
    """Pages and places in them of positions of slots."""
    page = s["case"]["page"]
    return s["pages"][slot, pos // page].long(), pos % page


def _plain_write(s, places, k, v):
    page, at = places
    for kind, x in enumerate((k, v)):
        code, scale = _plain_quantise(x)
        s["codes"][page, kind, :, at] = code[..., 0::2] | (code[..., 1::2] << 4)
        s["scales"][page, kind, :, at] = scale


def _plain_read(s, places, kind):
    """[rows][kv_heads][dim] in fp32"""
    page, at = places
    return _plain_values(s["codes"][page, kind, :, at], s["scales"][page, kind, :, at])


def _plain_store(s):
    n = s["case"]["tokens"]
    first, slots = s["offsets"][:-1].long(), s["slots"].long()
    seq = torch.repeat_interleave(torch.arange(len(slots), device="cuda"),
                                  s["offsets"][1:].long() - first, output_size=n)
    pos = s["before"][slots].long()[seq] + torch.arange(n, device="cuda") - first[seq]
    places = _plain_places(s, slots[seq], pos)
    _plain_write(s, places, s["k"][:n], s["v"][:n])
    for kind, out in enumerate((s["k_out"], s["v_out"])):
        out[:n] = _plain_read(s, places, kind).to(out.dtype)
    return {"k": s["k_out"], "v": s["v_out"]}


def _plain_attend(s):
    case, first = s["case"], 0
    rep = case["heads"] // case["kv_heads"]
    for i, (n, past) in enumerate(zip(s["rows"], s["past"])):
        places = _plain_places(s, s["slots_list"][i], torch.arange(past + n, device="cuda"))
        k, v = _plain_read(s, places, 0), _plain_read(s, places, 1)
        for a in range(0, n, 1024):
            b = min(a + 1024, n)
            rows = slice(first + a, first + b)
            q = s["q"][rows].float() * case["dim"] ** -0.5
            seen = past + b
            late = torch.arange(seen, device="cuda") > torch.arange(past + a, seen,
                                                                    device="cuda")[:, None]
            for h in range(case["kv_heads"]):
                heads = slice(h * rep, (h + 1) * rep)
                z = q[:, heads].transpose(0, 1) @ k[:seen, h].T
                z = z.masked_fill(late, -math.inf)
                p = (z - z.amax(-1, keepdim=True)).exp()
                o = (p @ v[:seen, h]) / p.sum(-1, keepdim=True)
                if case["gate"]:
                    o = o * torch.sigmoid(s["gate"][rows, heads].float()).transpose(0, 1)
                s["o"][rows, heads] = o.transpose(0, 1).to(s["o"].dtype)
        first += n
    return s["o"]


def _plain_linear(s):
    case = s["case"]
    scale = s["scales"].float().view(case["n"], -1, 1)
    w = (s["q"].view(case["n"], -1, case["group"]).float() * scale).bfloat16().float()
    y = s["x"].float() @ w.view(case["n"], case["k"]).T
    if case["bias"]:
        y = y + s["bias"]
    return y.to(TYPES[case["out"]])


# ---- in 64 bits, from the definitions -------------------------------------------
def _exact_held(x):
    """What a cache holds of rows [..., dim]."""
    x = x.double().unflatten(-1, (-1, 32))
    most = x.abs().amax(-1, keepdim=True)
    unit = torch.full_like(most, 2.0 ** -120)
    low = torch.log2(most.clamp(min=2.0 ** -126) / 7).ceil().clamp(-120, 125)
    for step in (1, 0, -1):  # the smallest of three neighbours that is large enough
        u = torch.exp2((low + step).clamp(-120, 125))
        unit = torch.where(most <= 7 * u, u, unit)
    y = (x / unit).abs()
    best, held = torch.full_like(y, math.inf), torch.zeros_like(y)
    for v in (0, 1, 2, 4, 0.5, 1.5, 3, 6):  # those of even codes first: they take the ties
        off = (y - v).abs()
        held = torch.where(off < best, torch.full_like(y, v), held)
        best = torch.minimum(best, off)
    return (held * unit * x.sign()).flatten(-2)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "linear":
        q = s["packed"]
        q = torch.stack([q & 15, q >> 4], 1).flatten().double()
        q = torch.where(q > 7, q - 16, q).view(case["n"], -1, case["group"])
        w = (q * s["scales"].double().view(case["n"], -1, 1)).float().bfloat16().double()
        y = s["x"].double() @ w.view(case["n"], case["k"]).T
        return y if s["bias"] is None else y + s["bias"].double()
    if case["op"] == "store":
        k, v = s["k_out"].double(), s["v_out"].double()
        n = case["tokens"]
        k[:n], v[:n] = _exact_held(s["k"][:n]), _exact_held(s["v"][:n])
        return {"k": k, "v": v}
    rep = case["heads"] // case["kv_heads"]
    o, row = s["o"].double(), 0
    for n, past, c in zip(s["rows"], s["past"], s["context"]):
        for h in range(case["kv_heads"]):
            k, v = _exact_held(c[0][:, h]), _exact_held(c[1][:, h])
            for a in range(0, n, 512):
                m = min(512, n - a)
                here = slice(row + a, row + a + m)
                for j in range(h * rep, (h + 1) * rep):
                    z = (s["q"][here, j].double() @ k[:past + a + m].T) / math.sqrt(case["dim"])
                    z = z + torch.full_like(z, -math.inf).triu(past + a + 1)
                    r = torch.softmax(z, -1) @ v[:past + a + m]
                    if case["gate"]:
                        r = r / (1 + (-s["gate"][here, j].double()).exp())
                    o[here, j] = r
        row += n
    return o


# ---- what a pass cannot do without ----------------------------------------------
def work(case):
    t = SIZE[case["type"]]
    if case["op"] == "linear":
        n, k, rows = case["n"], case["k"], case["rows"]
        return {"bytes": n * k // 2 + n * k // case["group"] * 2 + 4 * n * case["bias"]
                + rows * k * t + rows * n * SIZE[case["out"]], "flops": 2 * rows * n * k}
    rows, past = _lengths(case)
    h, d = case["kv_heads"], case["dim"]
    marks = 4 * (3 * case["seqs"] + 1)
    if case["op"] == "store":
        one = 2 * h * d
        return {"bytes": case["tokens"] * (one * t * 2 + (one // 2 + one // 32) * 2) + marks,
                "flops": 4 * case["tokens"] * one}
    held = sum(a + b for a, b in zip(rows, past))
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(rows, past))
    return {"bytes": held * 2 * h * (d // 2 + d // 32) + marks
            + case["tokens"] * case["heads"] * d * t * (2 + case["gate"]),
            "flops": 4 * pairs * case["heads"] * d}
