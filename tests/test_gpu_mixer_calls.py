"""The token mixer's calls at the edges of what they take: device batches whose offsets
fall between skipped sequences, the port block beside torch's streams and captured, a
layer that is refused, the most rows, a layer on host arrays."""
import pytest
import torch

import mixer_ref as R
from dismoen import DismoenError, GatedDelta, SeqBatch, ShortConv

pytestmark = pytest.mark.gpu


def rand(g, *shape, t=torch.float32):
    return torch.randn(shape, generator=g).to(t).cuda()


@pytest.mark.parametrize("op", ["conv", "delta"])
@pytest.mark.parametrize("off,slots,lost", [
    ([0, 9, 2, 4, 20], [0, -1, -1, 1], 3),
    ([0, 60, 2, 4, 70], [0, -1, -1, 1], 3),               # as chunks
    ([5, 30, 10, *[12] * 20, 40], [3, *[-1] * 21, 1], 22),  # behind many
    ([0, 9, 2, *[9] * 40, 15], [2, *[-7] * 41, 0], None),   # the least of them does not count
    ([0, 0, 7, *[3] * 9, 40], [2, -1, *[-1] * 9, 0], 11),
    ([4, *[8] * 30, 2, 50], [-1] * 30 + [-2, 0], 31),       # no sequence before it
], ids=str)
def test_offsets_that_fall_between_skipped_sequences(block, op, off, slots, lost):
    """A sequence before which some offset lies behind its first row is left out and
    reported, whoever's offset that is, as the host finds it."""
    assert len(off) == len(slots) + 1
    g = torch.Generator().manual_seed(len(off))
    rows, n = 96, 4
    batch = SeqBatch(torch.tensor(off, dtype=torch.int32).cuda(), rows, 75, n,
                     slots=torch.tensor(slots, dtype=torch.int32).cuda())
    if op == "conv":
        x, w = rand(g, rows, 64), rand(g, 64, 4)
        state, y = rand(g, n, 3, 64), rand(g, rows, 64)
        f, args = ShortConv(block, w), (x, state, batch, y)
        ref = lambda: R.conv(x, w, None, old, off, keep)[:2]  # noqa: E731
    else:
        q, k, v = rand(g, rows, 1, 64), rand(g, rows, 1, 64), rand(g, rows, 2, 64)
        a, b = -rand(g, rows, 2).abs(), rand(g, rows, 2).sigmoid()
        state, y = rand(g, n, 2, 64, 64), rand(g, rows, 2, 64)
        f, args = GatedDelta(block, 1, 2, 64, 64), (q, k, v, a, b, state, batch, y)
        ref = lambda: R.delta(q, k, v, a, b, old, off, keep)[:2]  # noqa: E731
    old, before = state.clone(), y.clone()
    torch.cuda.synchronize()
    f(*args)
    if lost is None:
        block.sync()
    else:
        with pytest.raises(DismoenError, match=f"sequence {lost}: offsets") as e:
            block.sync()
        assert e.value.code == 1
    keep = [-1 if i == lost else s for i, s in enumerate(slots)]
    want, new = ref()
    live = ~want.isnan().flatten(1).any(1)
    assert (y.cpu()[live].double() - want[live]).abs().max().item() < 1e-4 if live.any() else True
    assert torch.equal(y.cpu()[~live], before.cpu()[~live])
    assert (state.cpu().double() - new).abs().max() < 1e-4
    for i in set(range(n)) - set(keep):
        assert torch.equal(state[i], old[i])


def port_block(blk, rows=9):
    from dismoen import PortBlock, synth
    layer = synth.make_layer(**synth.CONFIG_TOY, seed=3)
    blk.upload_layer(0, layer)
    g = torch.Generator().manual_seed(rows)
    h = layer.hidden
    x, w = rand(g, rows, h), rand(g, h, 2 * h) * h ** -0.5
    port = PortBlock(blk, 0, 1 + 0.1 * rand(g, h), 1 + 0.1 * rand(g, h))
    arrays = [torch.zeros_like(x) for _ in range(3)]

    def mix(v):
        return (v @ w)[:, ::2].bfloat16().contiguous()

    def want():  # everything in order by waiting for the device
        def waited(v):
            torch.cuda.synchronize()
            out = mix(v)
            torch.cuda.synchronize()
            return out

        torch.cuda.synchronize()
        port(x, waited, *arrays)
        torch.cuda.synchronize()
        return [a.clone() for a in arrays]

    return port, x, mix, arrays, want


@pytest.mark.parametrize("view", [True, False])
def test_port_block_and_torch_streams(view):
    """On the block's own stream, with both streams busy: x, the mixer and y are in the
    order of torch's current stream, and what the mixer returned is not reused before
    the block has read it."""
    from dismoen import MoEBlock
    with MoEBlock(0) as blk:
        port, x, mix, arrays, want = port_block(blk)
        right = want()
        busy = torch.randn(2048, 2048, device="cuda")
        ours = torch.cuda.ExternalStream(blk.stream())
        source = x.clone()

        def work():
            for _ in range(20):
                torch.mm(busy, busy)

        def slow(v):
            out = mix(v)
            work()
            # (rows in another order of memory: the block takes a copy of them)
            return out.clone() if view else out.unflatten(0, (3, 3)).permute(1, 0, 2) \
                .contiguous().permute(1, 0, 2)

        for other in (False, True):
            stream = torch.cuda.Stream() if other else torch.cuda.current_stream()
            for a in (x, *arrays):
                a.zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(ours):
                work()
            with torch.cuda.stream(stream):
                work()
                x.copy_(source)
                y = port(x, slow, *arrays)
                junk = [torch.full((9, x.shape[1]), float("nan"), dtype=torch.bfloat16,
                                   device="cuda") for _ in range(8)]
                got = [a.clone() for a in arrays]
            torch.cuda.synchronize()
            blk.sync()
            assert y is arrays[2] and junk[0].isnan().all()
            for a, b in zip(got, right):
                assert torch.equal(a, b)


def test_port_block_captured():
    """A capture of torch's stream takes in the block's own one."""
    from dismoen import MoEBlock
    with MoEBlock(0) as blk:
        port, x, mix, arrays, want = port_block(blk)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        values = [x.clone(), x * 0.5 + 1, x.flip(0)]
        right = []
        for v in values:
            x.copy_(v)
            right.append(want())
        with torch.cuda.stream(stream):  # (buffers of its sizes, libraries' handles)
            port(x, mix, *arrays)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            port(x, mix, *arrays)
        for _ in range(2):
            for v, r in zip(values, right):
                x.copy_(v)
                for a in arrays:
                    a.zero_()
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                for a, b in zip(arrays, r):
                    assert torch.equal(a, b)
                blk.sync()
        del graph


def test_mixer_layer_refused_in_a_capture_changes_nothing():
    """The layer's delta rule needs memory that a capture cannot make: none of the three
    operators is recorded, and after a call of its sizes all are."""
    from dismoen import GatedDeltaMixer, MoEBlock
    g = torch.Generator().manual_seed(5)
    t, (hk, hv, dk, dv), rows = torch.bfloat16, (1, 2, 64, 64), 70
    ch = 2 * hk * dk + hv * dv
    with MoEBlock(0) as blk:
        mixer = GatedDeltaMixer(blk, hk, hv, dk, dv, rand(g, ch, 4), rand(g, hv), rand(g, hv),
                                rand(g, dv))
        off = torch.tensor([0, 20, 70], dtype=torch.int32).cuda()
        batch = SeqBatch(off, rows, 50, 2)
        mixed, z = rand(g, rows, ch, t=t), rand(g, rows, hv, dv, t=t)
        a, b = rand(g, rows, hv, t=t), rand(g, rows, hv, t=t)
        start = rand(g, 2, 3, ch, t=t), rand(g, 2, hv, dk, dv)
        cs, st = start[0].clone(), start[1].clone()
        work, out = torch.zeros_like(mixed), torch.zeros_like(z)
        args = (mixed, z, b, a, cs, st, batch, work, out)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        mark = torch.zeros(1, device="cuda")
        torch.cuda.synchronize()
        blk.set_stream(stream.cuda_stream)
        with torch.cuda.graph(graph, stream=stream):
            with pytest.raises(DismoenError, match="before the capture"):
                mixer(*args)
            mark.add_(1)
        blk.set_stream(None)
        # and one that the library refuses: its output on the gates
        with pytest.raises(DismoenError, match="overlap"):
            mixer(mixed, z, b, out[:, 0, :hv], *args[4:])
        blk.sync()
        graph.replay()
        torch.cuda.synchronize()
        assert mark.item() == 1 and not work.any() and not out.any()
        assert torch.equal(cs, start[0]) and torch.equal(st, start[1])
        mixer(*args)
        blk.sync()
        want = [x.clone() for x in (out, cs, st)]
        graph = torch.cuda.CUDAGraph()
        blk.set_stream(stream.cuda_stream)
        with torch.cuda.graph(graph, stream=stream):
            mixer(*args)
        blk.set_stream(None)
        for _ in range(3):
            cs.copy_(start[0])
            st.copy_(start[1])
            out.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip((out, cs, st), want):
                assert torch.equal(x, y)
        blk.sync()
        del graph


def test_conv_of_the_most_rows(block):
    """2^30 - 1 rows, which take more than one launch: offsets in elements and bytes are
    past 2^32, and the rows where a launch ends belong to a sequence that goes on."""
    rows, ch, t = (1 << 30) - 1, 5, torch.float16
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 25 GB")
    g = torch.Generator().manual_seed(30)
    x = torch.empty(rows, ch, dtype=t, device="cuda")
    y = torch.full_like(x, 7.0)
    w = rand(g, ch, 4)
    cuts = [0, 3, 1 << 20, (1 << 29) - 2, rows - 2]
    spots = [0, 1 << 20, (1 << 29) - 70, rows - 150]  # rows looked at
    part = rand(g, 150, ch, t=t)
    x.zero_()
    for at in spots:
        x[at:at + 150] = part
    start = rand(g, 4, 3, ch, t=t)
    state = start.clone()
    batch = SeqBatch(torch.tensor(cuts, dtype=torch.int32).cuda(), rows, rows, 4)
    torch.cuda.synchronize()
    ShortConv(block, w)(x, state, batch, y)
    block.sync()
    for at in spots:
        lo = max(0, at - 3)
        off = sorted({0, *(min(max(c - lo, 0), at + 150 - lo) for c in cuts)})
        first = next(i for i in range(4) if cuts[i + 1] > lo)
        # (the state of the first sequence here: its own, or the rows before)
        old = torch.zeros(len(off) - 1, 3, ch, dtype=t)
        for i in range(len(off) - 1):
            seq = first + i
            if seq < 4:
                old[i] = start[seq].cpu() if cuts[seq] >= lo else \
                    x[lo - 3:lo].cpu() if lo >= 3 and cuts[seq] <= lo - 3 else 0
        want, _, size = R.conv(x[lo:at + 150], w, None, old, off)
        inside = [r for r in range(at, at + 150) if r < cuts[4]]
        R.close(y[inside], want[[r - lo for r in inside]], size[[r - lo for r in inside]], 12)
    assert (y[cuts[4]:] == 7).all()
    for i in range(4):
        line = torch.cat([start[i], x[max(cuts[i], cuts[i + 1] - 3):cuts[i + 1]]])
        assert torch.equal(state[i], line[-3:])
    del x, y
    torch.cuda.empty_cache()


def test_mixer_layer_on_host_arrays(block):
    """The layer on numpy arrays gives the device tensors' bits, and leaves what is
    behind total_tokens."""
    from dismoen import GatedDeltaMixer
    g = torch.Generator().manual_seed(8)
    (hk, hv, dk, dv), rows = (1, 2, 64, 64), 60
    ch = 2 * hk * dk + hv * dv
    p = [rand(g, ch, 4), rand(g, hv), rand(g, hv), rand(g, dv)]
    ins = [rand(g, rows + 4, ch), rand(g, rows + 4, hv, dv), rand(g, rows, hv), rand(g, rows, hv)]
    cs, st = rand(g, 3, 3, ch), rand(g, 3, hv, dk, dv)
    work, out = torch.full((rows + 4, ch), 3.0).cuda(), torch.full((rows + 4, hv, dv), 3.0).cuda()
    off = torch.tensor([0, 1, 40, 60], dtype=torch.int32)
    host = [x.cpu().numpy().copy() for x in (*ins, cs, st)]
    hwork, hout = work.cpu().numpy().copy(), out.cpu().numpy().copy()
    torch.cuda.synchronize()
    GatedDeltaMixer(block, hk, hv, dk, dv, *p)(*ins, cs, st, SeqBatch(off.cuda(), rows, 39, 3),
                                               work, out)
    block.sync()
    GatedDeltaMixer(block, hk, hv, dk, dv, *(x.cpu().numpy() for x in p))(
        *host, SeqBatch(off.numpy(), rows, 39, 3), hwork, hout)
    for a, b in ((out, hout), (work, hwork), (cs, host[4]), (st, host[5])):
        assert torch.equal(a.cpu(), torch.from_numpy(b))
    assert (hout[rows:] == 3).all() and (hwork[rows:] == 3).all()
