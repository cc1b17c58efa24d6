"""Calls of the 4-bit cache and of attention at the edges of what they take: values that are
not finite where a row must not see them, device batches and pages that are wrong, captured
calls and their replays, host arrays, caches past 4 GB, a whole layer in a port block."""
import numpy as np
import pytest
import torch

import cache_ref as R
import mixer_ref as M
from dismoen import (AttentionMixer, CacheAttention, DismoenError, GatedNorm, KVCache, MoEBlock,
                     PortBlock, QuantLinear, SeqBatch, synth)
from test_gpu_cache import STEPS, TYPES, Cache, gen, rand, run
from test_gpu_linear import weights

pytestmark = pytest.mark.gpu


# ---- what a row does not see ----------------------------------------------------------------
@pytest.mark.parametrize("dim", [32, 96, 128, 256])
@pytest.mark.parametrize("past,rows", [([40, 3], [1, 2]), ([0, 130], [90, 70]), ([300], [5])])
def test_not_finite_behind_a_row(block, dim, past, rows):
    """Keys and values that are not finite reach the rows that see them, in the elements of
    their blocks, and no others."""
    def spoil(ctx):
        for c in ctx:
            n = c.shape[1]
            c[1, n - 1, 0, 3] = float("inf")          # a value that only the last row sees
            c[0, n - 1, 1, dim - 1] = float("nan")    # its key, of the other head
            if n > 60:
                c[1, 55, 1, dim - 2] = float("nan")   # one in the middle
    run(block, past, rows, 4, 2, dim, 16, torch.bfloat16, spoil=spoil)


def test_queries_that_are_not_finite(block):
    """They make their own rows NaN, and no other's."""
    g = gen("queries")
    for rows, heads in (([1, 1, 2], 8), ([70], 4)):
        c = Cache(block, g, [30] * len(rows), rows, 2, 64, 16)
        c.fill(block, [torch.randn((2, 30 + n, 2, 64), generator=g).cuda() for n in rows])
        q = rand(g, sum(rows), heads, 64)
        bad = q.clone()
        bad[0, 1, 5], bad[-1, heads - 1, 0] = float("nan"), float("inf")
        a, b = torch.empty_like(q), torch.empty_like(q)
        torch.cuda.synchronize()
        att = CacheAttention(block, heads)
        att(q, c.cache, c.batch(), a)
        att(bad, c.cache, c.batch(), b)
        block.sync()
        hit = torch.zeros(q.shape[:2], dtype=torch.bool)
        hit[0, 1] = hit[-1, heads - 1] = True
        assert b.cpu()[hit].isnan().all() and torch.equal(a.cpu()[~hit], b.cpu()[~hit])


@pytest.mark.parametrize("size,scale", [(1e-6, None), (60.0, None), (1.0, 1e-20), (1e-3, 1e4)])
def test_scores_of_all_sizes(block, size, scale):
    """Rows of even and of single probabilities."""
    run(block, [200, 3], [1, 40], 4, 2, 64, 16, torch.float32, size=size, scale=scale)


# ---- wrong device batches -----------------------------------------------------------------------
def test_sequences_that_are_left_out(block):
    g = gen("left out")
    heads, dim = 2, 64
    c = Cache(block, g, [20, 20, 20, 20, 20], [2, 3, 70, 1, 2], heads, dim, 16)
    c.fill(block, [torch.randn((2, 20 + n, heads, dim), generator=g).cuda() for n in c.rows])
    rows = sum(c.rows)
    q, out = rand(g, rows, 4, dim), torch.empty(rows, 4, dim, device="cuda")
    att = CacheAttention(block, 4)
    torch.cuda.synchronize()
    att(q, c.cache, c.batch(), out)
    block.sync()
    right, off = out.clone(), [0, 2, 5, 75, 76, 78]
    k, v = rand(g, rows, heads, dim), rand(g, rows, heads, dim)
    pages, before = c.pages.clone(), c.before.clone()
    codes, scales = c.codes.clone(), c.scales.clone()
    slot = c.slots.tolist()

    def spoil(what, i):
        if what == "past":
            c.before[slot[i]] = -1
        elif what == "long":
            c.before[slot[i]] = 16 * pages.shape[1] - c.rows[i] + 1
        else:
            c.pages[slot[i], 1] = what

    for i in range(5):
        for what, text in (("past", "its tokens"), ("long", "its tokens"), (1 << 20, "a page outside"),
                           (-3, "a page outside")):
            for call in ("write", "read", "attend"):
                c.pages.copy_(pages)
                c.before.copy_(before)
                c.codes.copy_(codes)
                c.scales.copy_(scales)
                out.fill_(5.0)
                spoil(what, i)
                torch.cuda.synchronize()
                if call == "attend":
                    att(q, c.cache, c.batch(), out)
                elif call == "write":
                    c.cache.write(k, v, c.batch())
                else:
                    c.cache.read(k, v, c.batch())
                with pytest.raises(DismoenError, match=f"sequence {i}: {text}") as e:
                    block.sync()
                assert e.value.code == 1
                block.sync()  # reported once
                if call == "attend":
                    keep = [t for t in range(rows) if not off[i] <= t < off[i + 1]]
                    # (the division of the work, and with it the order of sums, may change)
                    assert (out[keep] - right[keep]).abs().max() < 1e-4
                    if what in ("past", "long"):
                        assert (out[off[i]:off[i + 1]] == 5).all()
    # a slot that two sequences with rows name: reported by the call that writes
    c.pages.copy_(pages)
    c.before.copy_(before)
    same = c.slots.clone()
    same[3] = same[1]
    b = c.batch(slots=same.cuda())
    torch.cuda.synchronize()
    att(q, c.cache, b, out)
    block.sync()
    c.cache.write(k, v, b)
    with pytest.raises(DismoenError, match="sequence 3: names the state"):
        block.sync()


def test_skipped_and_empty_sequences(block):
    """Negative slots and sequences without rows leave everything as it is, whatever their
    offsets, and offsets behind the last one that counts are not looked at."""
    g = gen("skipped")
    heads, dim = 2, 64
    c = Cache(block, g, [33, 5, 9], [1, 30, 2], heads, dim, 16)
    c.fill(block, [torch.randn((2, p + n, heads, dim), generator=g).cuda()
                   for p, n in zip(c.past, c.rows)])
    q = rand(g, 40, 4, dim)
    one, two = torch.full_like(q, 2.0), torch.full_like(q, 2.0)
    att = CacheAttention(block, 4)
    slots = c.slots.tolist()
    b = SeqBatch(R.i32([0, 1, 1, 31, 31, 33, -7, 99]), 40, 30, c.num_slots,
                 slots=R.i32([slots[0], -1, slots[1], slots[0], slots[2], -2, -1]))
    torch.cuda.synchronize()
    att(q, c.cache, c.batch(), one)
    att(q, c.cache, b, two)
    block.sync()
    assert (one - two).abs().max() < 1e-5 and (two[33:] == 2).all()
    codes = c.codes.clone()
    k, v = rand(g, 40, heads, dim), rand(g, 40, heads, dim)
    torch.cuda.synchronize()
    c.cache.write(k, v, b)
    block.sync()
    first = c.codes.clone()
    c.codes.copy_(codes)
    torch.cuda.synchronize()
    c.cache.write(k, v, c.batch())
    block.sync()
    assert torch.equal(first, c.codes)


def test_thousands_of_sequences(block):
    """More sequences than any workgroup looks at at once, prompts among single tokens."""
    g = gen("thousands")
    n = 1300
    rows = [1] * n
    for i in range(7, n, 10):
        rows[i] = 17
    past = torch.randint(0, 40, (n,), generator=g).tolist()
    c = Cache(block, g, past, rows, 1, 32, 16)
    ctx = [torch.randn((2, a + b, 1, 32), generator=g).bfloat16() for a, b in zip(past, rows)]
    c.fill(block, [x.cuda() for x in ctx])
    q = rand(g, sum(rows), 4, 32, t=torch.bfloat16)
    o = torch.empty_like(q)
    torch.cuda.synchronize()
    CacheAttention(block, 4)(q, c.cache, c.batch(), o)
    block.sync()
    at = 0
    for i, m in enumerate(rows):
        if i % 97 == 7 or i % 211 == 0 or i in (255, 256, 511, 512, 1299):
            want, size = R.attend(q[at:at + m], R.held(ctx[i][0]), R.held(ctx[i][1]), past[i], 32 ** -0.5)
            M.close(o[at:at + m], want, size, STEPS[torch.bfloat16])
        at += m


def test_a_cache_past_4_gb(block):
    """Pages whose bytes lie behind 2^32, with scales and codes at their ends."""
    pages, page, heads, dim = 530, 16384, 2, 256
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 10 GB")
    g = gen("4 GB")
    cs, ss = KVCache.shapes(pages, heads, page, dim)
    codes = torch.zeros(cs, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(ss, dtype=torch.uint8, device="cuda")
    assert codes.numel() > 1 << 32
    ids = R.i32([[pages - 1, 3], [pages - 2, pages - 3]])
    past = R.i32([page - 5, 2 * page - 8])
    cache = KVCache(block, codes, scales, ids, past)
    k, v = rand(g, 15, heads, dim), rand(g, 15, heads, dim)
    b = SeqBatch(R.i32([0, 8, 15]), 15, 8, 2)
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    torch.cuda.synchronize()
    cache.write(k, v, b)
    cache.read(ko, vo, b)
    q = rand(g, 15, 4, dim)
    o = torch.empty_like(q)
    CacheAttention(block, 4)(q, cache, b, o)
    block.sync()
    assert torch.equal(ko.double().cpu(), R.held(k)) and torch.equal(vo.double().cpu(), R.held(v))
    # (zeros before: of keys and values)
    for s, lo, hi, before in ((0, 0, 8, page - 5), (1, 8, 15, 2 * page - 8)):
        zeros = torch.zeros(before, heads, dim, dtype=torch.float64)
        want, size = R.attend(q[lo:hi], torch.cat([zeros, R.held(k[lo:hi])]),
                              torch.cat([zeros, R.held(v[lo:hi])]), before, dim ** -0.5)
        M.close(o[lo:hi], want, size, 1024)
    del codes, scales
    torch.cuda.empty_cache()


# ---- captured ------------------------------------------------------------------------------------
@pytest.mark.parametrize("lens", [[1, 1, 1], [1, 90, 2]])
def test_captured(lens):
    """A captured step takes each replay's rows, slots, pages and past, and gives the bits of
    the same call made at once."""
    g = gen("captured", tuple(lens))
    heads, dim, qh = 2, 128, 8
    with MoEBlock(0) as blk:
        c = Cache(blk, g, [100, 40, 7], lens, heads, dim, 16, extra=8)
        c.fill(blk, [torch.randn((2, p + n, heads, dim), generator=g).cuda()
                     for p, n in zip(c.past, c.rows)])
        rows = sum(lens)
        k, v, q, out = (rand(g, rows, h, dim) for h in (heads, heads, qh, qh))
        mix, b = AttentionMixer(blk, qh), c.batch()
        start = c.codes.clone(), c.scales.clone()
        mark = torch.zeros(1, device="cuda")
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        blk.set_stream(stream.cuda_stream)
        with torch.cuda.graph(graph, stream=stream):  # no memory for it yet: nothing is recorded
            with pytest.raises(DismoenError, match="before the capture"):
                mix(q, k, v, c.cache, b, out)
            mark.add_(1)
        blk.set_stream(None)
        graph.replay()
        torch.cuda.synchronize()
        assert mark.item() == 1 and torch.equal(c.codes, start[0]) and torch.equal(c.scales, start[1])
        mix(q, k, v, c.cache, b, out)
        blk.sync()
        graph = torch.cuda.CUDAGraph()
        blk.set_stream(stream.cuda_stream)
        with torch.cuda.graph(graph, stream=stream):
            mix(q, k, v, c.cache, b, out)
        blk.set_stream(None)
        for i in range(4):
            # other rows, a shorter past and other pages
            for x in (k, v, q):
                x.copy_(rand(g, *x.shape))
            c.before[c.slots.long()] = torch.tensor([100 - 30 * i, 40 - i, 7 - 2 * i],
                                                    dtype=torch.int32, device="cuda")
            if i == 2:
                c.pages[c.slots[0].item(), :2] = c.pages[c.slots[0].item(), :2].flip(0)
            got = []
            for replay in (True, False):
                c.codes.copy_(start[0])
                c.scales.copy_(start[1])
                out.zero_()
                torch.cuda.synchronize()
                if replay:
                    graph.replay()
                else:
                    mix(q, k, v, c.cache, b, out)
                torch.cuda.synchronize()
                blk.sync()
                got.append((c.codes.clone(), c.scales.clone(), out.clone()))
            for x, y in zip(*got):
                assert torch.equal(x, y)
        del graph


def test_a_refused_layer_leaves_the_cache(block):
    g = gen("refused")
    c = Cache(block, g, [3], [4], 2, 64, 16)
    k, v, q = (rand(g, 4, h, 64) for h in (2, 2, 4))
    codes = c.codes.clone()
    mix = AttentionMixer(block, 4)
    torch.cuda.synchronize()
    for args, text in (((q, k, v, c.cache, c.batch(), q), "o must not overlap"),
                       ((q[:3], k, v, c.cache, c.batch(), torch.empty_like(q)), "fewer rows"),
                       ((q, k, v[:, :1], c.cache, c.batch(), torch.empty_like(q)), "2 heads of 64"),
                       ((q.half(), k, v, c.cache, c.batch(), torch.empty_like(q)), "heads of 64")):
        with pytest.raises(DismoenError, match=text):
            mix(*args)
    block.sync()
    assert torch.equal(codes, c.codes)
    with MoEBlock(0) as other:
        with pytest.raises(DismoenError, match="another block"):
            CacheAttention(other, 4)(q, c.cache, c.batch(), torch.empty_like(q))


# ---- host arrays ---------------------------------------------------------------------------------
def test_host_arrays(block):
    """numpy arrays give the device tensors' bits; outputs that lie between others leave those."""
    g = gen("host")
    heads, dim, qh = 2, 64, 4
    c = Cache(block, g, [20, 0, 5], [1, 70, 3], heads, dim, 16)
    rows = sum(c.rows)
    k, v = rand(g, rows, heads, dim), rand(g, rows, heads, dim)
    qg = rand(g, rows, qh, 2, dim)
    out = torch.empty(rows, qh, dim, device="cuda")
    c.fill(block, [torch.randn((2, p + n, heads, dim), generator=g).cuda()
                   for p, n in zip(c.past, c.rows)])
    host = KVCache(block, *(x.cpu().numpy().copy() for x in (c.codes, c.scales, c.pages, c.before)))
    off = np.array([0, 1, 71, 74], np.int32)
    hb = SeqBatch(off, rows, 70, c.num_slots, slots=c.slots.numpy())
    AttentionMixer(block, qh)(qg[:, :, 0], k, v, c.cache, c.batch(), out, gate=qg[:, :, 1])
    block.sync()
    hq = qg.cpu().numpy()
    wide = np.full((rows, qh, 2, dim), 3, np.float32)
    AttentionMixer(block, qh)(hq[:, :, 0], k.cpu().numpy(), v.cpu().numpy(), host, hb, wide[:, :, 0],
                              gate=hq[:, :, 1])
    assert np.array_equal(wide[:, :, 0], out.cpu().numpy()) and (wide[:, :, 1] == 3).all()
    assert np.array_equal(host.arrays[0], c.codes.cpu().numpy())
    assert np.array_equal(host.arrays[1], c.scales.cpu().numpy())
    both = np.full((rows, 2, heads, dim), 4, np.float32)
    host.read(both[:, 0], both[:, 1], hb)
    assert np.array_equal(both[:, 0], R.held(k).numpy()) and np.array_equal(both[:, 1], R.held(v).numpy())


# ---- together --------------------------------------------------------------------------------------
def test_full_attention_layer(block):
    """A full-attention layer of a port block: 4-bit projections, norms of queries and keys,
    the cache, gated attention, and the projection back, for two steps of a prompt and
    single tokens; against the same from the definitions in 64 bits."""
    g = gen("layer")
    with MoEBlock(0) as blk:
        layer = synth.make_layer(**synth.CONFIG_TOY, seed=5)
        blk.upload_layer(0, layer)
        hidden, qh, kh, d = layer.hidden, 4, 2, 64
        w_in, s_in, p_in = weights(g, (2 * qh + 2 * kh) * d, hidden, 32)
        w_out, s_out, p_out = weights(g, hidden, qh * d, 32)
        proj_in = QuantLinear(blk, w_in.shape[0], hidden, s_in.cuda(), p_in.cuda(), 32)
        proj_out = QuantLinear(blk, hidden, qh * d, s_out.cuda(), p_out.cuda(), 32)
        gq, gk = 1 + 0.1 * rand(g, d), 1 + 0.1 * rand(g, d)
        q_norm, k_norm = GatedNorm(blk, d, qh, gamma=gq), GatedNorm(blk, d, kh, gamma=gk)
        mixer, port = AttentionMixer(blk, qh), PortBlock(blk, 0)
        c = Cache(blk, g, [0, 0, 0], [23, 1, 2], kh, d, 16, extra=2)
        c.before.zero_()
        held = [[torch.zeros(0, kh, d, dtype=torch.float64)] * 2 for _ in range(3)]
        for lens in ([23, 1, 2], [1, 1, 1]):
            rows = sum(lens)
            x = rand(g, rows, hidden)
            batch = c.batch(lens)
            seen = {}

            def mix(xn):
                mid = torch.empty(rows, w_in.shape[0], device="cuda")
                proj_in(xn, mid)
                qg = mid[:, :2 * qh * d].unflatten(1, (qh, 2, d))
                k, v = mid[:, 2 * qh * d:].unflatten(1, (2, kh, d)).unbind(1)
                q = torch.empty(rows, qh, d, device="cuda")
                blk.sync()
                q.copy_(qg[:, :, 0])
                torch.cuda.synchronize()
                q_norm(q, stream=q)
                k_norm(k, stream=k)
                o = torch.empty(rows, qh, d, device="cuda")
                mixer(q, k, v, c.cache, batch, o, gate=qg[:, :, 1])
                out = torch.empty(rows, hidden, device="cuda")
                proj_out(o.flatten(1), out)
                blk.sync()
                seen.update(xn=xn.clone(), q=q, k=k, v=v, o=o, out=out, gate=qg[:, :, 1])
                return out

            arrays = [torch.empty(rows, hidden, device="cuda") for _ in range(3)]
            torch.cuda.synchronize()
            port(x, mix, *arrays)
            torch.cuda.synchronize()
            blk.sync()
            # each step from what went into it
            mid = seen["xn"].double().cpu() @ w_in.T
            size = seen["xn"].double().cpu().abs() @ w_in.abs().T
            M.close(seen["v"], mid[:, (2 * qh + kh) * d:].unflatten(1, (kh, d)),
                    size[:, (2 * qh + kh) * d:].unflatten(1, (kh, d)), 64)
            at = 0
            for i, n in enumerate(lens):
                before = held[i][0].shape[0]
                held[i] = [torch.cat([h, R.held(seen[key][at:at + n])])
                           for h, key in zip(held[i], "kv")]
                want, size = R.attend(seen["q"][at:at + n], *held[i], before, d ** -0.5,
                                      seen["gate"][at:at + n])
                M.close(seen["o"][at:at + n], want, size, STEPS[torch.float32])
                at += n
            o = seen["o"].flatten(1).double().cpu()
            M.close(seen["out"], o @ w_out.T, o.abs() @ w_out.abs().T, 64)
            assert arrays[2].isfinite().all()
            c.before[c.slots.long()] += torch.tensor(lens, dtype=torch.int32, device="cuda")


def test_on_torchs_stream():
    """On a stream of the caller's, behind and before other work on it."""
    g = gen("stream")
    with MoEBlock(0) as blk:
        c = Cache(blk, g, [50], [2], 2, 64, 16)
        c.fill(blk, [torch.randn((2, 52, 2, 64), generator=g).cuda()])
        lin_w, s, p = weights(g, 64, 256, 32)
        lin = QuantLinear(blk, 64, 256, s.cuda(), p.cuda(), 32)
        q0 = rand(g, 2, 4, 64)
        q, o, y = torch.zeros_like(q0), torch.zeros_like(q0), torch.zeros(2, 64, device="cuda")
        stream, busy = torch.cuda.Stream(), torch.randn(2048, 2048, device="cuda")
        torch.cuda.synchronize()
        blk.set_stream(stream.cuda_stream)
        with torch.cuda.stream(stream):
            for _ in range(20):
                torch.mm(busy, busy)
            q.copy_(q0)
            CacheAttention(blk, 4)(q, c.cache, c.batch(), o)
            lin(o.flatten(1), y)
            q.zero_()
            got = o.clone(), y.clone()
        torch.cuda.synchronize()
        q.copy_(q0)
        torch.cuda.synchronize()
        CacheAttention(blk, 4)(q, c.cache, c.batch(), o)
        lin(o.flatten(1), y)
        blk.sync()
        assert torch.equal(got[0], o) and torch.equal(got[1], y)
        blk.set_stream(None)
