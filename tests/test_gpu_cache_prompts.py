"""Attention of several prompts in one call, at all kinds of head ratios, against the
formula in 64 bits.

Tolerance, as in test_gpu_cache: half a step of the output's type, plus roundings of 2^-24 of
sum(p |v|) (1 + sum |q k| scale).  A score 50; the maximum's difference, the scale and
exp2 (1 ulp) 4; p's parts 1 for fp32 rows (2^-24) and 128 for those of 16 bits (2^-17).
Sums over a context of up to 2752 tokens: for every 32 of them one addition a part of p (two,
three in fp32) and half a factor, 86 * 2.5 = 215 and 86 * 3.5 = 301, and within the 32 another
6 + 2 of their own share.  Joining at most 8 parts 24, the quotient and the gate 8: 437 and
396."""
import pytest
import torch

import cache_ref as R
import mixer_ref as M
from dismoen import CacheAttention
from test_gpu_cache import TYPES, Cache, gen, rand

pytestmark = pytest.mark.gpu

STEPS = {torch.float32: 396, torch.float16: 437, torch.bfloat16: 437}
LONGEST = 2752


def attend(q, k, v, past, scale, gate=None):
    """cache_ref.attend for many rows, a head at a time on the GPU."""
    n, heads, _ = q.shape
    rep = heads // k.shape[1]
    q, k, v = q.double(), k.cuda(), v.cuda()
    o, size = torch.empty_like(q), torch.empty_like(q)
    late = torch.arange(past + n, device="cuda") > past + torch.arange(n, device="cuda")[:, None]
    for h in range(heads):
        kk, vv = k[:, h // rep].contiguous(), v[:, h // rep].contiguous()
        p = torch.softmax((scale * (q[:, h].contiguous() @ kk.T.contiguous())).masked_fill(late, -torch.inf), 1)
        terms = (q[:, h].abs().contiguous() @ kk.abs().T.contiguous()).masked_fill(late, 0).amax(1)
        o[:, h] = p @ vv
        size[:, h] = (p @ vv.abs()) * (1 + scale * terms[:, None])
    if gate is not None:
        g = torch.sigmoid(gate.double())
        o, size = o * g, size * g
    return o.cpu(), size.cpu()


def run(block, seqs, heads, kv_heads, dim, t, gate=False, page=16, skip=(), pad=3):
    """seqs: (rows, tokens before) of each; those in skip have a slot that leaves them out."""
    rows, past = [n for n, _ in seqs], [p for _, p in seqs]
    assert max(n + p for n, p in seqs) <= LONGEST
    g = gen("prompts", seqs, heads, dim)
    c = Cache(block, g, past, rows, kv_heads, dim, page)
    ctx = [torch.randn((2, p + n, kv_heads, dim), generator=g).to(t) for n, p in seqs]
    c.fill(block, [x.cuda() for x in ctx])
    total = sum(rows) + pad
    x = rand(g, total, heads, 2, dim, t=t)
    q, gates = x[:, :, 0], x[:, :, 1] if gate else None
    o = torch.full((total, heads, dim), float("nan"), dtype=t, device="cuda")
    slots = c.slots.clone()
    for i in skip:
        slots[i] = -1
    batch = c.batch(pad=pad, slots=slots.cuda())
    torch.cuda.synchronize()
    CacheAttention(block, heads)(q, c.cache, batch, o, gate=gates)
    block.sync()
    at = 0
    for i, n in enumerate(rows):
        got = o[at:at + n]
        if i in skip:
            assert got.isnan().all()
        elif n:
            want, size = attend(q[at:at + n], R.held(ctx[i][0]), R.held(ctx[i][1]), past[i], dim ** -0.5,
                                None if gates is None else gates[at:at + n])
            M.close(got, want, size, STEPS[t])
        at += n
    assert o[at:].isnan().all()


# (heads, key heads, dim): batches whose last tokens, rows or walk a division of the work in
# fractions would lose; then prompts with single tokens, empty and skipped ones between and
# behind them
BATCHES = [
    (40, 8, 128, [(700, 0), (700, 1000), (1000, 0)], ()),
    (28, 4, 128, [(256, 1000), (300, 500), (300, 100)], ()),
    (6, 1, 64, [(339, 1769), (530, 578), (741, 0)], ()),
    (12, 4, 256, [(148, 0), (306, 1288), (316, 0)], ()),
    (24, 4, 64, [(654, 381), (868, 99), (668, 1820), (1, 0), (897, 0), (1, 0)], ()),
    (24, 2, 32, [(1, 300), (500, 0), (0, 9), (2000, 700), (1, 0), (90, 31), (0, 0), (1, 2000)], ()),
    (9, 3, 96, [(300, 5), (200, 0), (1, 70), (400, 33), (64, 0), (150, 600), (3, 9)], (1, 6)),
    (14, 2, 192, [(129, 0), (1, 900), (333, 12), (1, 0), (700, 64), (2, 2)], (2,)),
    (8, 4, 128, [(1300, 0), (1, 20), (700, 700), (0, 0), (40, 5)], (1,)),
]


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,seqs,skip", BATCHES, ids=lambda v: str(v)[:24])
def test_prompts_together(block, heads, kv_heads, dim, seqs, skip, t):
    run(block, seqs, heads, kv_heads, dim, t, gate=dim < 128, skip=skip)


@pytest.mark.parametrize("ratio", [3, 5, 6, 7, 12])
@pytest.mark.parametrize("dim,t", [(64, torch.float32), (128, torch.float16), (256, torch.bfloat16)],
                         ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("num", [3, 20])
def test_ratios(block, ratio, dim, t, num):
    g = gen("ratios", ratio, dim, num)

    def pick(lo, hi):
        return int(torch.randint(lo, hi + 1, (1,), generator=g))
    most = 1800 // num
    seqs = [(pick(most // 3, most) if i % 3 != 1 else 1, pick(0, 1) * pick(1, 900)) for i in range(num)]
    run(block, seqs + [(1, 40)], 2 * ratio, 2, dim, t, page=64)


def test_many_prompts(block):
    """More sequences than a workgroup has threads, at a ratio that is no power of two."""
    g = gen("many prompts")
    rows = torch.randint(1, 50, (530,), generator=g).tolist()
    past = torch.randint(0, 60, (530,), generator=g).tolist()
    run(block, list(zip(rows, past)), 3, 1, 64, torch.bfloat16)
