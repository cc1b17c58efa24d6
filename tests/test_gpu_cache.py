"""The 4-bit cache and attention over it, against 64-bit restatements.

The cache's values are exact.  Tolerances of attention: half a step of the output's
type, plus roundings of 2^-24 of sum(p |v|) (1 + sum |q k| scale), the size that
cache_ref.attend gives: a score is a sum of up to 256 products, added 32 at a time
(8 sums of at most 6 roundings), scaled, and its maximum subtracted (2): 50 roundings of
its terms' size, each a relative error of p; exp2 is within 1 ulp, p's parts within 2^-17
for rows of 16 bits (2^7 roundings of 2^-24) and 2^-24 for fp32; sums over the context
are added by 32 tokens, a factor at each: 2 per step, of which lanes, waves and parts
share the tokens, 64 for the contexts here; the quotient and the gate 8."""
import zlib

import pytest
import torch

import cache_ref as R
import mixer_ref as M
from dismoen import CacheAttention, DismoenError, KVCache, SeqBatch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
STEPS = {torch.float32: 128, torch.float16: 256, torch.bfloat16: 256}


def gen(*seed):
    return torch.Generator().manual_seed(zlib.crc32(repr(seed).encode()))


def rand(g, *shape, t=torch.float32):
    return torch.randn(shape, generator=g).to(t).cuda()


class Cache:
    """A cache of slots with past tokens, their pages in a random order."""

    def __init__(self, blk, g, past, rows, heads, dim, page, spare=2, extra=1):
        self.n, self.past, self.rows = len(past), past, rows
        self.num_slots = self.n + spare
        need = [-(-(p + r) // page) for p, r in zip(past, rows)]
        num = sum(need) + 2
        ids = torch.randperm(num, generator=g).int()
        self.slots = torch.randperm(self.num_slots, generator=g)[:self.n].int()
        pages = torch.full((self.num_slots, max(1, *need) + extra), -5, dtype=torch.int32)
        before = torch.full((self.num_slots,), -7, dtype=torch.int32)
        at = 0
        for i, slot in enumerate(self.slots.tolist()):
            pages[slot, :need[i]] = ids[at:at + need[i]]
            before[slot] = past[i]
            at += need[i]
        self.codes = torch.randint(0, 256, (num, 2, heads, page, dim // 2), generator=g,
                                   dtype=torch.uint8).cuda()
        # (bytes of all values, NaN among them, wherever nothing is written)
        self.scales = torch.randint(0, 256, (num, 2, heads, page, dim // 32), generator=g,
                                    dtype=torch.uint8).cuda()
        self.scales[self.scales % 3 == 0] = 255
        self.pages, self.before = pages.cuda(), before.cuda()
        torch.cuda.synchronize()
        self.cache = KVCache(blk, self.codes, self.scales, self.pages, self.before)

    def batch(self, lens=None, fresh=None, pad=0, max_len=None, slots=None):
        lens = self.rows if lens is None else lens
        off = [0]
        for r in lens:
            off.append(off[-1] + r)
        return SeqBatch(R.i32(off), off[-1] + pad, max_len or max(1, *lens), self.num_slots,
                        slots=self.slots.cuda() if slots is None else slots,
                        fresh=None if fresh is None else R.i32(fresh))

    def fill(self, blk, contexts):
        """Every sequence's context [2][past + rows][heads][dim] into the cache."""
        b = self.batch([c.shape[1] for c in contexts], fresh=[1] * self.n)
        k, v = (torch.cat([c[i] for c in contexts]).contiguous() for i in (0, 1))
        torch.cuda.synchronize()
        self.cache.write(k, v, b)
        blk.sync()


# ---- the cache -------------------------------------------------------------------------
def spread(g, shape, t):
    """Rows whose blocks differ in size, with zeros, ties and largest elements among them."""
    x = torch.randn(shape, generator=g, dtype=torch.float64)
    blocks = x.unflatten(-1, (-1, 32))
    blocks *= torch.exp2(torch.randint(-9, 9, blocks.shape[:-1], generator=g)).unsqueeze(-1)
    kind = torch.rand(blocks.shape[:-1], generator=g)
    ties = torch.randint(-28, 29, blocks.shape, generator=g) / 4.0
    blocks[kind < 0.3] = ties[kind < 0.3].double()
    blocks[kind < 0.05] = 0
    return x.to(t)


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
def test_write_and_read(block, dim, t):
    """Rows of every head size come back as the values that the definition gives, all else
    in the cache and in the arrays read into stays."""
    g = gen("cache", dim)
    heads, page = 3, 16
    c = Cache(block, g, [0, 5, 31, 16, 100], [40, 1, 2, 16, 0], heads, dim, page)
    rows = sum(c.rows)
    k, v = (spread(g, (rows + 2, heads, dim), t).cuda() for _ in range(2))
    codes, scales = c.codes.clone(), c.scales.clone()
    torch.cuda.synchronize()
    c.cache.write(k, v, c.batch(pad=2))
    block.sync()
    ko, vo = (torch.full((rows + 2, heads, dim), 3.0, dtype=t, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    c.cache.read(ko, vo, c.batch(pad=2))
    block.sync()
    for got, x in ((ko, k), (vo, v)):
        assert torch.equal(got[:rows].double().cpu(), R.held(x[:rows]).to(t).double())
        assert (got[rows:] == 3).all()
    # pages that no row lies in, and the places in pages that none does
    touched = torch.zeros(c.codes.shape[0], dtype=torch.bool)
    for slot, past, n in zip(c.slots.tolist(), c.past, c.rows):
        for p in range(past, past + n):
            touched[c.pages[slot, p // page].item()] = True
    assert torch.equal(c.codes.cpu()[~touched], codes.cpu()[~touched])
    assert torch.equal(c.scales.cpu()[~touched], scales.cpu()[~touched])
    assert int((c.scales != scales).sum()) <= rows * 2 * heads * dim // 32


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("heads,more", [(1, 1.01), (5, 1.5), (3, 3.7)])
def test_many_rows_at_once(block, dim, t, heads, more):
    """Calls of several words a thread, of sequences that begin and end anywhere among four
    rows, hold what the definition gives, in rows with gaps between heads."""
    g = gen("at once", dim, heads)
    rows = int(more * 2 ** 20) // (heads * dim) + 3
    lens = [1, 2, 3, 0, 517, 5, rows - 528]
    c = Cache(block, g, [3, 0, 6, 9, 77, 2, 14], lens, heads, dim, 16)
    k, v = (torch.full((rows + 5, heads + 1, dim), 7.0, dtype=t, device="cuda") for _ in range(2))
    x = [spread(g, (rows, heads, dim), t) for _ in range(2)]
    k[:rows, :heads], v[:rows, 1:] = x[0].cuda(), x[1].cuda()
    out = [torch.full((rows + 5, heads + 1, dim), 3.0, dtype=t, device="cuda") for _ in range(2)]
    before = c.codes.clone()
    torch.cuda.synchronize()
    c.cache.write(k[:, :heads], v[:, 1:], c.batch(pad=5))
    c.cache.read(out[0][:, 1:], out[1][:, :heads], c.batch(pad=5))
    block.sync()
    for got, y in ((out[0][:, 1:], x[0]), (out[1][:, :heads], x[1])):
        assert torch.equal(got[:rows].double().cpu(), R.held(y).to(t).double())
    assert (out[0][:, 0] == 3).all() and (out[1][:, heads] == 3).all()
    assert all((o[rows:] == 3).all() for o in out)
    # rows of the pages in front of a sequence's and behind them stay
    for slot, past, n in zip(c.slots.tolist(), c.past, lens):
        for pos in (past - 1, past + n):
            if pos < 0 or pos >= -(-(past + n) // 16) * 16:
                continue
            page = c.pages[slot, pos // 16].item()
            # (a key's codes lie together, in the order of positions)
            assert torch.equal(c.codes[page, 0, :, pos % 16], before[page, 0, :, pos % 16])


@pytest.mark.parametrize("page", [16, 64, 1024])
def test_write_in_steps(block, page):
    """Rows written one by one and a few at a time give the bytes of one call."""
    g = gen("steps", page)
    heads, dim, n = 2, 128, 61
    k, v = rand(g, n, heads, dim, t=torch.bfloat16), rand(g, n, heads, dim, t=torch.bfloat16)
    whole = Cache(block, gen(page), [0], [n], heads, dim, page)
    parts = Cache(block, gen(page), [0], [n], heads, dim, page)
    whole.cache.write(k, v, whole.batch())
    at = 0
    for step in (1, 1, 3, 16, 1, 32, 7):
        parts.before[parts.slots.long()] = at
        torch.cuda.synchronize()
        parts.cache.write(k[at:at + step], v[at:at + step], parts.batch([step]))
        block.sync()
        at += step
    assert at == n
    assert torch.equal(whole.codes, parts.codes) and torch.equal(whole.scales, parts.scales)


def test_strided_rows_and_extremes(block):
    """Heads that lie apart in one projected row; the smallest and largest blocks, and
    blocks that are not finite."""
    g = gen("strided")
    heads, dim, rows = 2, 64, 9
    x = torch.randn((rows, heads, 3, dim), generator=g)
    x[0, 0, 0] *= 1e-38
    x[1, 0, 0] = 1.2e-37
    x[2, 1, 0] = torch.finfo(torch.float32).max
    x[3, 0, 1, 5] = float("inf")
    x[4, 1, 1, 40] = float("nan")
    x[5, 0, 2, 33] = -float("inf")
    x[6, 0, 2] = -0.0
    x[7, 1, 0] = 7.0
    x[8, 1, 0] = 7.0000005
    y = x.cuda()
    out = torch.zeros_like(y)
    c = Cache(block, g, [3], [rows], heads, dim, 16)
    for i, j in ((0, 1), (2, 1)):
        torch.cuda.synchronize()
        c.cache.write(y[:, :, i], y[:, :, j], c.batch())
        c.cache.read(out[:, :, i], out[:, :, 1], c.batch())
        block.sync()
        for n in (i, j):
            want = R.held(x[:, :, n])
            got = out[:, :, n].double().cpu()
            assert torch.equal(got.isnan(), want.isnan())
            assert torch.equal(got.nan_to_num(nan=9.0), want.nan_to_num(nan=9.0))


# ---- attention ---------------------------------------------------------------------------
def run(block, past, rows, heads, kv_heads, dim, page, t, gate=True, pad=2, size=1.0, scale=None,
        spoil=None):
    g = gen("attend", tuple(past), tuple(rows), heads, dim, page)
    c = Cache(block, g, past, rows, kv_heads, dim, page)
    ctx = [torch.randn((2, a + b, kv_heads, dim), generator=g) for a, b in zip(past, rows)]
    if spoil:
        spoil(ctx)
    ctx = [x.to(t) for x in ctx]
    c.fill(block, [x.cuda() for x in ctx])
    total = sum(rows) + pad
    x = rand(g, total, heads, 2, dim, t=t) * size
    q, gates = x[:, :, 0], x[:, :, 1] if gate else None
    o = rand(g, total, heads, dim, t=t)
    before = o.clone()
    torch.cuda.synchronize()
    CacheAttention(block, heads, scale)(q, c.cache, c.batch(pad=pad), o, gate=gates)
    block.sync()
    at = 0
    for i, n in enumerate(rows):
        if n:
            k, v = R.held(ctx[i][0]), R.held(ctx[i][1])
            want, sz = R.attend(q[at:at + n], k, v, past[i], scale or dim ** -0.5,
                                None if gates is None else gates[at:at + n])
            got = o[at:at + n]
            assert torch.equal(got.isnan().cpu(), want.isnan())
            # A probability enters as bf16 parts, which end at 2^-126: what lies below, in each
            # of up to three parts and in the exponential itself, is 0 instead, at most
            # 4 * 2^-126 of each token's value (as many roundings of 2^-24 as STEPS of it).
            lost = v.shape[0] * 2.0 ** -124 * v.nan_to_num(nan=0.0).abs().max() / STEPS[t] * 2.0 ** 24
            M.close(got.nan_to_num(nan=1.0), want.nan_to_num(nan=1.0),
                    sz.nan_to_num(nan=1.0) + lost, STEPS[t])
        at += n
    assert torch.equal(o[at:], before[at:])
    return c, q, gates, o


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
def test_single_tokens(block, dim, t):
    run(block, [0, 1, 15, 16, 31, 32, 33, 127, 128, 129, 700], [1] * 11, 4, 2, dim, 16, t)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (16, 2), (16, 1), (17, 1), (40, 1),
                                            (66, 1), (96, 1), (5, 5)])
def test_heads(block, heads, kv_heads):
    run(block, [40, 200], [1, 2], heads, kv_heads, 64, 32, torch.bfloat16)


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
def test_prompts(block, dim, t):
    run(block, [0, 50, 0, 17], [70, 33, 1, 40], 6, 2, dim, 16, t, gate=False)


@pytest.mark.parametrize("rows", [2, 3, 8, 9, 16, 17, 31, 32, 33, 63, 64, 65, 129])
@pytest.mark.parametrize("past", [0, 95])
def test_row_counts(block, rows, past):
    run(block, [past], [rows], 4, 2, 128, 64, torch.float16)


def test_one_long_context(block):
    """A context over many workgroups, and one that ends in a tile's first token."""
    run(block, [9000], [1], 8, 1, 128, 256, torch.bfloat16)
    run(block, [8192], [1], 4, 4, 64, 16, torch.float32, gate=False)
    run(block, [5000], [3], 8, 2, 256, 64, torch.bfloat16)


def test_many_sequences(block):
    """More sequences than a workgroup has threads, skipped and empty ones among them."""
    g = gen("many")
    past = torch.randint(0, 70, (600,), generator=g).tolist()
    rows = torch.randint(0, 3, (600,), generator=g).tolist()
    rows[300] = 80
    run(block, past, rows, 2, 1, 32, 16, torch.bfloat16)
