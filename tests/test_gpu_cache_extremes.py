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
