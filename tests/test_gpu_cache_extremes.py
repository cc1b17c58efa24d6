"""Attention with queries and scores at the ends of fp32, against the formula in 64 bits.
Tolerances are those of test_gpu_cache."""
import pytest
import torch

import cache_ref as R
import mixer_ref as M
from dismoen import CacheAttention
from test_gpu_cache import STEPS, Cache, gen

pytestmark = pytest.mark.gpu


def attend(block, past, rows, heads, kv_heads, dim, t, scale, q, ctx):
    """(result, definition, size, what is held) of each sequence."""
    g = gen("extremes", tuple(past), tuple(rows), dim)
    c = Cache(block, g, past, rows, kv_heads, dim, 16)
    ctx = [x.to(t) for x in ctx]
    c.fill(block, [x.cuda() for x in ctx])
    q = q.to(t).cuda()
    o = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    CacheAttention(block, heads, scale)(q, c.cache, c.batch(), o)
    block.sync()
    at = 0
    for i, n in enumerate(rows):
        k, v = R.held(ctx[i][0]), R.held(ctx[i][1])
        want, size = R.attend(q[at:at + n], k, v, past[i], scale)
        yield o[at:at + n], want, size, q[at:at + n], k, v
        at += n


@pytest.mark.parametrize("dim", [32, 128, 256])
@pytest.mark.parametrize("past,rows", [([40, 3, 0], [1, 2, 1]), ([0, 130], [90, 70])])
def test_largest_queries(block, dim, past, rows):
    """fp32 queries above bf16's largest value: every bit of them counts, none overflows."""
    g = gen("largest", dim, sum(rows))
    most = torch.finfo(torch.float32).max
    q = torch.rand((sum(rows), 6, dim), generator=g) * 0.01 + 0.99
    q = q * most * torch.where(torch.rand(q.shape, generator=g) < 0.5, -1.0, 1.0)
    q[0] = most
    # keys of 2^-100: scores of some 2^128 * 2^-100 * sqrt(dim)
    ctx = [torch.randn((2, p + n, 2, dim), generator=g) for p, n in zip(past, rows)]
    for x in ctx:
        x[0] *= 2.0 ** -100
    scale = 2.0 ** -28 * dim ** -0.5
    for got, want, size, *_ in attend(block, past, rows, 6, 2, dim, torch.float32, scale, q, ctx):
        assert got.isfinite().all()
        M.close(got, want, size, STEPS[torch.float32])


@pytest.mark.parametrize("t", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [2.0 ** 31, 1e12, 1e29, 1e30])
@pytest.mark.parametrize("past,rows", [([0, 2, 0, 700], [1, 1, 2, 1]), ([0, 31], [150, 90])])
def test_large_scores(block, past, rows, scale, t):
    """Scores of 2^31 and more, where their rounding alone is more than fp32's exponents: a row is
    the value of its largest score.  Some rows see negative scores alone."""
    dim = 64
    g = gen("scores", sum(rows), scale)
    q = torch.randn((sum(rows), 6, dim), generator=g)
    q[:, 1] = -q[:, 1].abs()
    ctx = [torch.randn((2, p + n, 2, dim), generator=g) for p, n in zip(past, rows)]
    for x in ctx:
        x[0, :, 0] = x[0, :, 0].abs() + 0.5  # keys of query heads 0 to 2
    at = 0
    for i, (got, _, _, q, k, v) in enumerate(attend(block, past, rows, 6, 2, dim, t, scale, q, ctx)):
        for r in range(rows[i]):
            z = torch.einsum("hd,jhd->hj", q[r].double().cpu(),
                             k[:past[i] + r + 1].repeat_interleave(3, 1))
            top = z.topk(min(2, z.shape[1]), 1)
            # two scores' errors, of 50 roundings of their terms each, must not change which is
            # larger, and the difference has to leave nothing of the other's probability
            terms = torch.einsum("hd,jhd->hj", q[r].double().cpu().abs(),
                                 k[:past[i] + r + 1].abs().repeat_interleave(3, 1)).amax(1)
            clear = torch.ones(6, dtype=torch.bool)
            if z.shape[1] > 1:
                gap = top.values[:, 0] - top.values[:, 1]
                clear = gap > 100 * 2.0 ** -24 * terms + 2.0 ** 8 / scale
            at += int(clear.sum())
            want = v[top.indices[:, 0], torch.arange(6) // 3]
            assert torch.equal(got[r].double().cpu()[clear], want.to(t).double()[clear])
    assert at > 6 * sum(rows) * 0.95
