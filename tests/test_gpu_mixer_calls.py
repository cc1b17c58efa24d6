"""The token mixer's calls at the edges of what they take: device batches whose offsets
fall between skipped sequences."""
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
