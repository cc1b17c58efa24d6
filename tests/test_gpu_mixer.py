"""The token mixer's kernels against 64-bit restatements.

Tolerances: half a step of the output's type, plus roundings of 2^-24 of the
sizes that are summed.
  convolution  at most 4 products and a bias (5 roundings), SiLU from the
               hardware's exp2 and reciprocal (each within 1 ulp, its argument
               within 2: 6 more, on a value no larger than the sum): 12
  norms        a sum of up to 8192 squares in 32 per lane and 8 halvings (40
               roundings, halved by the root), divide, root and four products:
               32; a gate adds the 6 of SiLU
  delta rule   per row: sums of up to 32 terms per lane and three halvings (35),
               norms and gates (below 20), the update (3): 64 of the largest
               column norm, and a row never enlarges an earlier error (the
               state's factor exp(g) (I - beta k k^T) has norm 1 at most), so
               64 per row of a sequence's length"""
import zlib

import numpy as np
import pytest
import torch

import mixer_ref as R
from dismoen import DismoenError, GatedDelta, GatedDeltaMixer, GatedNorm, SeqBatch, ShortConv

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROUNDINGS = {"conv": 12, "norm": 40, "delta": 64}


def rand(g, *shape, t=torch.float32):
    return torch.randn(shape, generator=g).to(t).cuda()


def gen(*seed):
    return torch.Generator().manual_seed(zlib.crc32(repr(seed).encode()))


class Seqs:
    """Sequences of the given lengths from row `at` on, with slots in another
    order and one slot to spare per sequence."""

    def __init__(self, lens, g, pad=3, skip=(), fresh=True, max_len=None):
        off = np.cumsum([0, *lens]).astype(np.int32)
        self.n, self.rows, self.lens = len(lens), int(off[-1]) + pad, lens
        self.num_slots = 2 * self.n
        self.slots = torch.randperm(self.num_slots, generator=g)[: self.n].int()
        for i in skip:
            self.slots[i] = -1 - i
        self.fresh = (torch.rand(self.n, generator=g) < 0.4).int() if fresh else None
        self.off = torch.from_numpy(off)
        self.batch = SeqBatch(self.off.cuda(), self.rows, max_len or max(1, *lens), self.num_slots,
                              slots=self.slots.cuda(),
                              fresh=None if self.fresh is None else self.fresh.cuda())
        self.args = (self.off, self.slots, self.fresh)


def check_rows(got, want, scale, steps, before):
    """Rows of a sequence are right, the others are what they were."""
    none = want.isnan().flatten(1).any(1)
    assert torch.equal(got[none.to(got.device)], before[none.to(got.device)])
    scale = scale[~none] if isinstance(scale, torch.Tensor) and scale.shape[0] == want.shape[0] \
        else scale
    R.close(got[~none.to(got.device)], want[~none], scale, steps)


LENS = [[1], [1, 1, 1, 1, 1], [0, 1, 2, 3, 4, 5, 0], [40], [17, 0, 1, 33, 2], [300, 3, 70]]


# ---- short convolution --------------------------------------------------------------
def run_conv(block, lens, channels, width, t, bias=True, silu=True, x_pitch=0, y_pitch=0, skip=(),
             shift=0):
    g = gen("conv", tuple(lens), channels, width)
    s = Seqs(lens, g, skip=skip)
    x = rand(g, s.rows, channels + x_pitch, t=t)[:, shift: shift + channels]
    y = rand(g, s.rows, channels + y_pitch, t=t)
    w = rand(g, channels, width)
    b = rand(g, channels) if bias else None
    state = rand(g, s.num_slots, width - 1, channels, t=t)
    before, old = y.clone(), state.clone()
    torch.cuda.synchronize()
    ShortConv(block, w, bias=b, silu=silu)(x, state, s.batch, y[:, :channels])
    block.sync()
    want, new, size = R.conv(x, w, b, old, *s.args, silu=silu)
    check_rows(y[:, :channels], want, size, ROUNDINGS["conv"], before[:, :channels])
    assert torch.equal(y[:, channels:], before[:, channels:])
    assert torch.equal(state.cpu(), new.to(t))  # rows as they came, bit for bit
    return x, y, state


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_conv(block, lens, width, t):
    run_conv(block, lens, 520, width, t)


@pytest.mark.parametrize("channels,x_pitch,y_pitch,shift,t", [
    (1, 0, 0, 0, "bf16"), (7, 0, 0, 0, "f16"), (64, 3, 0, 0, "bf16"), (64, 8, 16, 8, "bf16"),
    (64, 8, 8, 1, "f16"), (2049, 0, 5, 0, "f32"), (8192, 0, 0, 0, "bf16"), (257, 0, 0, 0, "f32"),
])
def test_conv_layouts(block, channels, x_pitch, y_pitch, shift, t):
    run_conv(block, [5, 0, 1, 30], channels, 4, TYPES[t], bias=False, x_pitch=x_pitch,
             y_pitch=y_pitch, shift=shift)


def test_conv_many_rows(block):
    """Tiles of 16 rows, sequences that begin one, two and three rows before a
    tile's end, single rows in a row, and skipped ones."""
    lens = [13, 3, 14, 2, 15, 1, 16, 31, 1, 1, 1, 1, 30, 0, 2, 2, 700]
    run_conv(block, lens, 4096, 4, torch.bfloat16, skip=(1, 8))
    run_conv(block, lens, 4096, 4, torch.bfloat16, silu=False)


def test_conv_continues(block):
    """A sequence in two calls gives the bits of one call."""
    g = gen("continues")
    x, w = rand(g, 50, 96, t=torch.bfloat16), rand(g, 96, 4)
    op = ShortConv(block, w)
    for cut in (1, 2, 3, 16, 49):
        state = torch.zeros(1, 3, 96, dtype=torch.bfloat16, device="cuda")
        one, two = torch.empty_like(x), torch.empty_like(x)
        whole = state.clone()
        torch.cuda.synchronize()
        off = [torch.tensor(o, dtype=torch.int32, device="cuda") for o in ([0, 50], [0, cut],
                                                                          [0, 50 - cut])]
        torch.cuda.synchronize()
        op(x, whole, SeqBatch(off[0], 50, 50, 1), one)
        op(x[:cut], state, SeqBatch(off[1], cut, 50, 1), two[:cut])
        op(x[cut:], state, SeqBatch(off[2], 50 - cut, 50, 1), two[cut:])
        block.sync()
        assert torch.equal(one, two) and torch.equal(whole, state)


# ---- norms ----------------------------------------------------------------------------
def run_norm(block, rows, groups, dim, t, st, post=True, gamma=True, act="silu", residual=True,
             vec=False, edge=True, stream=True, pitch=0, scale=0.5, size=1.0):
    g = gen("norm", rows, groups, dim, act, residual)
    w = groups * dim

    def array(ty, p=pitch):
        return (rand(g, rows, w + p) * size).to(ty)[:, p:].unflatten(1, (groups, dim))

    x = array(t)
    gate = array(t) if act else None
    res = array(st) if residual else None
    gm = rand(g, dim) if gamma and post else None
    em = rand(g, dim) if gamma and edge else None
    sc = rand(g, groups, dim) if vec else scale
    out = torch.full((rows, w + pitch), 7.0, dtype=st, device="cuda")
    y = torch.full((rows, w + pitch), 7.0, dtype=st, device="cuda")
    ov, yv = (a[:, pitch:].unflatten(1, (groups, dim)) for a in (out, y))
    op = GatedNorm(block, dim, groups, gamma=gm, edge_gamma=em, post=post, edge=edge, gate=act,
                   scale=sc)
    torch.cuda.synchronize()
    op(x, ov if stream else None, yv if edge else None, gate=gate, residual=res)
    block.sync()
    want, want_y, terms = R.norm(x, gm, post, gate, act, res, sc, em)
    assert (out[:, :pitch] == 7).all() and (y[:, :pitch] == 7).all()
    if stream:
        R.close(ov, want, terms, ROUNDINGS["norm"])
    else:
        assert (out == 7).all()
    if edge:
        # the stream's roundings, divided as the stream is, besides y's own
        root = (want.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        e = 1.0 if em is None else em.double().cpu().abs()
        rms = (terms.square().mean(-1, keepdim=True)).sqrt()
        R.close(yv, want_y, terms / root * e + want_y.abs() * rms / root, ROUNDINGS["norm"])


@pytest.mark.parametrize("dim", [1, 7, 8, 64, 65, 128, 130, 136, 512, 513, 520, 2048, 2049, 2056,
                                 4096, 5001, 8192, 8191])
@pytest.mark.parametrize("t,st", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32"), ("f16", "f16"),
                                  ("f32", "f32")])
def test_norm_dims(block, dim, t, st):
    run_norm(block, 5, 1, dim, TYPES[t], TYPES[st])


@pytest.mark.parametrize("kw", [
    dict(act=None), dict(act="sigmoid"), dict(post=False), dict(post=False, act=None),
    dict(residual=False), dict(residual=False, edge=False), dict(vec=True), dict(stream=False),
    dict(gamma=False), dict(edge=False, vec=True), dict(pitch=8), dict(pitch=3), dict(scale=-2.5),
    dict(size=1e-4), dict(size=100.0),
], ids=str)
@pytest.mark.parametrize("rows,groups,dim", [(1, 1, 2048), (37, 3, 40), (3, 32, 128), (9, 2, 33)])
def test_norm_options(block, rows, groups, dim, kw):
    run_norm(block, rows, groups, dim, torch.bfloat16, torch.float32, **kw)


def test_norm_many_rows(block):
    run_norm(block, 70001, 1, 16, torch.bfloat16, torch.bfloat16)


@pytest.mark.parametrize("dim", [60, 96, 128, 130, 255, 260, 512])
def test_norm_of_many_rows_is_that_of_few(block, dim):
    """Many rows take half the lanes a row: the same sums, and right."""
    rows = (1 << 21) // dim + 5
    run_norm(block, rows, 1, dim, torch.bfloat16, torch.float32, residual=False)
    g = gen("many", dim)
    x, z, r = (rand(g, rows, 1, dim) for _ in range(3))
    op = GatedNorm(block, dim, gate="silu", edge=True)
    torch.cuda.synchronize()
    many = op(x, torch.empty_like(x), torch.empty_like(x), gate=z, residual=r)
    few = op(x[:9], torch.empty_like(x[:9]), torch.empty_like(x[:9]), gate=z[:9], residual=r[:9])
    block.sync()
    assert torch.equal(many[0][:9], few[0]) and torch.equal(many[1][:9], few[1])


def test_norm_in_place_and_special_values(block):
    g = gen("place")
    x, z, r = (rand(g, 6, 1, 64) for _ in range(3))
    z[0, 0, :5] = torch.tensor([200.0, -200.0, 3e38, -3e38, 0.0])
    x[1] = 0  # a row of zeros: rmsnorm gives zeros, not NaN
    x[2, 0, 3] = float("inf")
    x[3, 0, 3] = float("nan")
    z[4, 0, 7] = float("inf")
    op = GatedNorm(block, 64, gate="silu", edge=False)
    plain = torch.empty_like(x)
    on_res, on_x = r.clone(), x.clone()
    torch.cuda.synchronize()
    op(x, plain, gate=z, residual=r)
    op(x, on_res, gate=z, residual=on_res)
    op(on_x, on_x, gate=z, residual=r)
    block.sync()
    same = lambda a, b: torch.equal(a.nan_to_num(1.5, 2.5, 3.5), b.nan_to_num(1.5, 2.5, 3.5))  # noqa: E731
    assert same(plain, on_res) and same(plain, on_x)
    want, _, terms = R.norm(x, None, True, z, "silu", r)
    fine = want.isfinite()
    assert torch.equal(plain.cpu().isfinite(), fine)
    R.close(plain.cpu()[fine], want[fine], terms[fine], ROUNDINGS["norm"])
    assert torch.equal(plain[1].cpu(), r[1].cpu())


# ---- the gated delta rule ---------------------------------------------------------------
def delta_inputs(g, rows, hk, hv, dk, dv, t, raw=True, pitch=0, shift=0):
    kw, vw = hk * dk, hv * dv
    x = torch.randn((rows, 2 * kw + vw + pitch), generator=g)
    x = (x * torch.sigmoid(x)).to(t).cuda()[:, shift:]
    q = x[:, :kw].unflatten(1, (hk, dk))
    k = x[:, kw:2 * kw].unflatten(1, (hk, dk))
    v = x[:, 2 * kw:2 * kw + vw].unflatten(1, (hv, dv))
    if raw:
        a, b = rand(g, rows, hv, t=t), rand(g, rows, hv, t=t)
        gates = {"a_log": rand(g, hv), "dt_bias": rand(g, hv) - 2}
    else:
        a, b = -torch.rand((rows, hv), generator=g).cuda(), torch.rand((rows, hv), generator=g).cuda()
        gates = {"a_log": None, "dt_bias": None}
    return q, k, v, a, b, gates


def run_delta(block, lens, hk, hv, dk, dv, t, raw=True, qk_norm=True, pitch=0, shift=0, skip=(),
              change=None, scale=None):
    g = gen("delta", tuple(lens), hk, hv, dk, dv)
    s = Seqs(lens, g, skip=skip)
    q, k, v, a, b, gates = delta_inputs(g, s.rows, hk, hv, dk, dv, t, raw, pitch, shift)
    if not qk_norm:
        q, k = q * 0.1, (k.float() / (k.float().norm(dim=-1, keepdim=True) + 0.1)).to(t)
    if change:
        change(q, k, v, a, b, gates)
    state = rand(g, s.num_slots, hv, dk, dv) * 0.3
    o = rand(g, s.rows, hv, dv, t=t)
    before, old = o.clone(), state.clone()
    op = GatedDelta(block, hk, hv, dk, dv, qk_norm=qk_norm, scale=scale, **gates)
    torch.cuda.synchronize()
    op(q, k, v, a, b, state, s.batch, o)
    block.sync()
    want, new, largest = R.delta(q, k, v, a, b, old, *s.args, **gates, qk_norm=qk_norm, scale=scale)
    n = max(1, *lens) * ROUNDINGS["delta"]
    m = float(largest.max())
    qsize = dk ** -0.5 if scale is None else abs(scale)
    if not qk_norm:
        qsize *= float(q.float().norm(dim=-1).max())
    check_rows(o, want, m * qsize, n, before)
    R.close(state, new, m, n)
    touched = {slot for _, _, _, slot, _ in R.seqs_of(*s.args, s.num_slots)}
    for i in range(s.num_slots):
        if i not in touched:
            assert torch.equal(state[i], old[i])
    return s, (q, k, v, a, b), old, state, o, op


SHAPES = [(1, 1, 128, 128), (2, 6, 128, 128), (2, 4, 64, 64), (3, 3, 8, 8), (1, 2, 72, 40),
          (1, 2, 256, 256), (2, 2, 136, 24), (1, 3, 64, 200)]
DELTA_LENS = [[1], [1] * 7, [0, 1, 2, 3, 0, 9], [32, 31, 1], [33, 64, 65, 2], [63, 127, 128, 129],
              [300, 5, 40]]


@pytest.mark.parametrize("lens", DELTA_LENS, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_delta(block, shape, lens):
    run_delta(block, lens, *shape, torch.bfloat16)


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("lens", [[1, 1, 1], [20, 1], [100, 64, 0, 3]], ids=str)
@pytest.mark.parametrize("kw", [
    dict(), dict(raw=False), dict(qk_norm=False), dict(pitch=8), dict(pitch=3),
    dict(pitch=9, shift=1), dict(skip=(0,)), dict(scale=-3.0)], ids=str)
def test_delta_options(block, kw, lens, t):
    run_delta(block, lens, 2, 4, 64, 96, t, **kw)


def _set(**kw):
    def change(q, k, v, a, b, gates):
        for name, value in kw.items():
            {"q": q, "k": k, "v": v, "a": a, "b": b}[name].copy_(
                value if isinstance(value, torch.Tensor) else torch.tensor(value))
    return change


@pytest.mark.parametrize("lens", [[5], [150, 7]], ids=str)
@pytest.mark.parametrize("raw,change", [
    (False, _set(a=0.0, b=1.0)),             # nothing decays, every row replaces in full
    (False, _set(a=0.0, b=0.0)),             # nothing is written
    (False, _set(a=-float("inf"), b=0.7)),   # every row forgets all before it
    (False, _set(a=-50.0, b=0.3)), (False, _set(a=-1e30, b=1.0)),
    (False, _set(a=-1e-7, b=2.0)),           # reflections
    (True, _set(a=80.0, b=90.0)), (True, _set(a=-90.0, b=-90.0)),
    (True, _set(q=0.0)), (True, _set(k=0.0)), (True, _set(v=0.0)),
    (True, _set(k=1.0)),                     # one key over and over
    (False, lambda q, k, v, a, b, gates: (k.fill_(1.0), a.fill_(0.0), b.fill_(1.0))),
])
def test_delta_gates_and_keys(block, lens, raw, change):
    run_delta(block, lens, 1, 2, 64, 64, torch.float32, raw=raw, change=change)


def test_delta_forgets_in_the_middle(block):
    def change(q, k, v, a, b, gates):
        a[::17] = -float("inf")
        a[5::23] = -300.0
    run_delta(block, [200, 30], 1, 2, 64, 64, torch.float32, raw=False, change=change)


def test_delta_sequences_are_alone(block):
    """A sequence's bits are the same whatever else is in the call."""
    lens = [1, 70, 0, 32, 200, 33, 1]
    s, ins, old, state, o, op = run_delta(block, lens, 2, 4, 128, 128, torch.bfloat16)
    for i, n in enumerate(lens):
        if not n:
            continue
        at = int(s.off[i])
        alone = torch.zeros_like(o[at: at + n])
        st = old[int(s.slots[i])][None].clone()
        fresh = s.fresh[i: i + 1].cuda()
        off = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        op(*(x[at: at + n] for x in ins), st, SeqBatch(off, n, n + 1000, 1, fresh=fresh), alone)
        block.sync()
        assert torch.equal(alone, o[at: at + n]) and torch.equal(st[0], state[int(s.slots[i])])


def test_delta_twice_the_same(block):
    first = run_delta(block, [90, 1, 260], 2, 4, 64, 64, torch.bfloat16)
    again = run_delta(block, [90, 1, 260], 2, 4, 64, 64, torch.bfloat16)
    assert torch.equal(first[3], again[3]) and torch.equal(first[4], again[4])


def test_delta_bad_values_stay_in_their_sequence(block):
    g = gen("nan")
    lens = [100, 64, 3, 90, 2]
    s = Seqs(lens, g, fresh=False)
    q, k, v, a, b, gates = delta_inputs(g, s.rows, 1, 2, 64, 64, torch.bfloat16)
    op = GatedDelta(block, 1, 2, 64, 64, **gates)
    start = rand(g, s.num_slots, 2, 64, 64)
    outs = []
    for bad in (False, True):
        if bad:
            k[int(s.off[1]) + 10, 0, 3] = float("nan")
            v[int(s.off[3]) + 70, 1, 3] = float("inf")
            a[int(s.off[4]) + 1, 0] = float("nan")
            q[s.rows - 3:] = float("nan")  # rows behind the last sequence
        state, o = start.clone(), torch.zeros_like(v)
        torch.cuda.synchronize()
        op(q, k, v, a, b, state, s.batch, o)
        block.sync()
        outs.append((state, o))
    (s0, o0), (s1, o1) = outs
    off = s.off.tolist()
    for i in (0, 2):
        slot = int(s.slots[i])
        assert torch.equal(s0[slot], s1[slot])
        assert torch.equal(o0[off[i]:off[i + 1]], o1[off[i]:off[i + 1]])
    assert s1[int(s.slots[1])].isnan().all()
    # the other head of a sequence, and rows more than 63 before, are untouched
    assert torch.equal(s0[int(s.slots[3]), 0], s1[int(s.slots[3]), 0])
    assert torch.equal(o0[off[3]:off[3] + 7], o1[off[3]:off[3] + 7])
    assert not s1[int(s.slots[3]), 1, :, 3].isfinite().any()
    assert s1[int(s.slots[4]), 0].isnan().all() and torch.equal(s0[int(s.slots[4]), 1],
                                                               s1[int(s.slots[4]), 1])


# ---- what the device finds wrong with the sequences ---------------------------------------
@pytest.mark.parametrize("op", ["conv", "delta"])
@pytest.mark.parametrize("off,slots,text,lost", [
    ([0, 4, 2, 80], [0, 1, 2], "sequence 1: offsets", (1, 2)),  # (2's rows are partly 0's)
    ([-3, 4, 9, 80], [0, 1, 2], "sequence 0: offsets", (0,)),
    ([0, 9, 4, 50], [0, -1, 2], "sequence 2: offsets", (2,)),  # rows of sequence 0, behind a skipped one
    ([0, 9, 0, 0], [0, -1, -1], None, ()),  # padding
    ([0, 4, 9, 2000000000], [0, 1, 2], "sequence 2: offsets", (2,)),
    ([0, 4, 9, 90], [0, 1, 2], "sequence 2: longer", (2,)),
    ([0, 4, 9, 80], [0, 6, 2], "sequence 1: slot outside", (1,)),
    ([0, 4, 9, 80], [0, 2000000000, 2], "sequence 1: slot outside", (1,)),
    ([0, 4, 9, 80], [3, 1, 3], "sequence 2: names the state", (0, 2)),
    ([0, 4, 9, 9], [3, 1, 3], None, ()),
    ([0, 4, 4, 79], [1, 1, 3], None, ()),
    ([0, 4, 9, 80], [3, -2, 5], None, ()),
])
def test_bad_sequences(block, op, off, slots, text, lost):
    g = gen("bad", op)
    rows, n = 96, 6
    o = torch.tensor(off, dtype=torch.int32).cuda()
    sl = torch.tensor(slots, dtype=torch.int32).cuda()
    batch = SeqBatch(o, rows, 75, n, slots=sl)
    if op == "conv":
        x, w = rand(g, rows, 64), rand(g, 64, 4)
        state, y = rand(g, n, 3, 64), rand(g, rows, 64)
        f = ShortConv(block, w)
        args = (x, state, batch, y)
        ref = lambda: R.conv(x, w, None, old, off, slots)[:2]  # noqa: E731
    else:
        q, k, v, a, b, gates = delta_inputs(g, rows, 1, 2, 64, 64, torch.float32)
        state, y = rand(g, n, 2, 64, 64), rand(g, rows, 2, 64)
        f = GatedDelta(block, 1, 2, 64, 64, **gates)
        args = (q, k, v, a, b, state, batch, y)
        ref = lambda: R.delta(q, k, v, a, b, old, off, slots, **gates)[:2]  # noqa: E731
    old, before = state.clone(), y.clone()
    torch.cuda.synchronize()
    f(*args)
    if text is None:
        block.sync()
    else:
        with pytest.raises(DismoenError, match="SEQUENCE_ERROR") as e:
            block.sync()
        assert text in str(e.value) and e.value.code == 1
        block.sync()  # reported once
    # the right ones are right, whatever the others are
    good = [i for i in range(3) if i not in lost and slots[i] >= 0]
    keep = [-1 if i not in good else s for i, s in enumerate(slots)]
    slots = keep
    want, new = ref()
    for i in good:
        b, e = off[i], off[i + 1]
        if e > b:
            assert (y[b:e].cpu().double() - want[b:e]).abs().max() < 1e-4
            assert (state[keep[i]].cpu().double() - new[keep[i]]).abs().max() < 1e-4
    if not lost:
        for i in range(n):
            if i not in keep:
                assert torch.equal(state[i], old[i])
    assert torch.equal(y[90:], before[90:])


# ---- host arrays, streams, graphs ----------------------------------------------------------
def to_np(t):
    t = t.cpu().contiguous()
    return R.bf16_bits(t).copy() if t.dtype == torch.bfloat16 else t.numpy().copy()


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES)
def test_host_arrays_give_the_same_bits(block, t):
    g = gen("host")
    lens = [3, 0, 90, 1]
    s = Seqs(lens, g)
    hb = SeqBatch(s.off.numpy(), s.rows, max(lens), s.num_slots, slots=s.slots.numpy(),
                  fresh=s.fresh.numpy())
    x, w, bias = rand(g, s.rows, 40, t=t), rand(g, 40, 4), rand(g, 40)
    state, y = rand(g, s.num_slots, 3, 40, t=t), rand(g, s.rows, 40, t=t)
    hx, hs, hy = to_np(x), to_np(state), to_np(y)
    ShortConv(block, to_np(w), bias=to_np(bias))(hx, hs, hb, hy)
    torch.cuda.synchronize()
    ShortConv(block, w, bias=bias)(x, state, s.batch, y)
    block.sync()
    assert np.array_equal(hy, to_np(y)) and np.array_equal(hs, to_np(state))

    q, k, v, a, b, gates = delta_inputs(g, s.rows, 1, 2, 64, 32, t)
    state, o = rand(g, s.num_slots, 2, 64, 32), rand(g, s.rows, 2, 32, t=t)
    ha = [to_np(z) for z in (q, k, v, a, b, state)]
    ho = to_np(o)
    GatedDelta(block, 1, 2, 64, 32, **{n: to_np(z) for n, z in gates.items()})(*ha, hb, ho)
    torch.cuda.synchronize()
    GatedDelta(block, 1, 2, 64, 32, **gates)(q, k, v, a, b, state, s.batch, o)
    block.sync()
    assert np.array_equal(ho, to_np(o)) and np.array_equal(ha[5], to_np(state))

    x, r = rand(g, 9, 2, 48, t=t), rand(g, 9, 2, 48)
    out, y, gm = torch.empty_like(r), torch.empty_like(r), rand(g, 48)
    hout, hy = to_np(out), to_np(y)
    GatedNorm(block, 48, 2, gamma=to_np(gm), edge=True)(to_np(x), hout, hy, residual=to_np(r))
    torch.cuda.synchronize()
    GatedNorm(block, 48, 2, gamma=gm, edge=True)(x, out, y, residual=r)
    block.sync()
    assert np.array_equal(hout, to_np(out)) and np.array_equal(hy, to_np(y))


def test_host_outputs_side_by_side(block):
    """Two outputs that are columns of one host buffer, and rows with something
    else between them: neither takes back what lies between its rows."""
    g = gen("side")
    x, gm = rand(g, 9, 2, 48), rand(g, 48)
    both = np.full((9, 3, 2, 48), 7.0, np.float32)
    norm = GatedNorm(block, 48, 2, gamma=to_np(gm), edge=True)
    norm(to_np(x), both[:, 0], both[:, 2])
    apart = [np.zeros((9, 2, 48), np.float32) for _ in range(2)]
    norm(to_np(x), *apart)
    assert np.array_equal(both[:, 0], apart[0]) and np.array_equal(both[:, 2], apart[1])
    assert (both[:, 1] == 7.0).all()


def test_calls_without_rows(block):
    """Empty tensors, which have no address."""
    e = torch.empty(0, 2, 48, device="cuda")
    GatedNorm(block, 48, 2, edge=True, gate="silu")(e, e, e, gate=e)
    g = gen("empty")
    mixer, p, ch = mixer_layer(block, g)
    t = torch.bfloat16
    cs, st = rand(g, 3, 3, ch, t=t), rand(g, 3, 4, 64, 64)
    before = cs.clone(), st.clone()
    s = SeqBatch(torch.zeros(3, dtype=torch.int32, device="cuda"), 0, 1, 3)
    r = lambda *d: torch.empty(0, *d, dtype=t, device="cuda")
    mixer(r(ch), r(4, 64), r(4), r(4), cs, st, s, r(ch), r(4, 64))
    block.sync()
    assert torch.equal(cs, before[0]) and torch.equal(st, before[1])


def mixer_layer(block, g, hk=2, hv=4, dk=64, dv=64, t=torch.bfloat16):
    ch = 2 * hk * dk + hv * dv
    p = {"conv_weight": rand(g, ch, 4) * 0.5, "a_log": rand(g, hv), "dt_bias": rand(g, hv) - 2,
         "norm_gamma": 1 + 0.1 * rand(g, dv)}
    return GatedDeltaMixer(block, hk, hv, dk, dv, **p), p, ch


def mixer_ref(p, mixed, z, b, a, conv_state, state, seqs, hk, hv, dk, dv, t):
    """The three operators in 64 bits, each one's rows rounded to their type."""
    y, cs, _ = R.conv(mixed, p["conv_weight"], None, conv_state, *seqs)
    y = y.to(t).double()
    n, kw = y.shape[0], hk * dk
    o, st, _ = R.delta(y[:, :kw].reshape(n, hk, dk), y[:, kw:2 * kw].reshape(n, hk, dk),
                       y[:, 2 * kw:].reshape(n, hv, dv), a, b, state, *seqs, a_log=p["a_log"],
                       dt_bias=p["dt_bias"])
    return R.norm(o.to(t).double(), p["norm_gamma"], True, z, "silu")[0], cs, st


@pytest.mark.parametrize("lens", [[1, 1, 1], [150, 1, 0, 20]], ids=str)
def test_mixer_layer(block, lens):
    """The three operators as a layer runs them; a rounding of one that falls on
    the other side than the reference's moves what follows by a step of bf16, so
    the whole is held to 2^-6 of its size in the 2-norm."""
    g = gen("layer")
    t, dims = torch.bfloat16, (2, 4, 64, 64)
    mixer, p, ch = mixer_layer(block, g, *dims)
    s = Seqs(lens, g)
    mixed, z = rand(g, s.rows, ch, t=t), rand(g, s.rows, 4, 64, t=t)
    a, b = rand(g, s.rows, 4, t=t), rand(g, s.rows, 4, t=t)
    cs, st = rand(g, s.num_slots, 3, ch, t=t), rand(g, s.num_slots, 4, 64, 64) * 0.1
    cs0, st0 = cs.clone(), st.clone()
    work, out = torch.empty_like(mixed), torch.empty_like(z)
    torch.cuda.synchronize()
    mixer(mixed, z, b, a, cs, st, s.batch, work, out)
    block.sync()
    want, wcs, wst = mixer_ref(p, mixed, z, b, a, cs0, st0, s.args, *dims, t)
    n = int(s.off[-1])
    assert torch.equal(cs.cpu(), wcs.to(t))
    for got, ref in ((out[:n], want[:n]), (st, wst)):
        d = (got.cpu().double() - ref).norm() / ref.norm()
        assert d < 2.0 ** -6, float(d)


def test_mixer_on_another_stream_captured_and_replayed(block):
    """One step captured on the caller's stream; replays take the rows, offsets,
    slots and states of the moment, with eager calls of more rows between them,
    which outgrow the buffers that the graph holds."""
    g = gen("graph")
    t, dims = torch.bfloat16, (1, 2, 64, 64)
    mixer, p, ch = mixer_layer(block, g, *dims)
    rows, n = 120, 8

    def fresh_step(seed, cuts):
        g = gen("step", seed)
        off = torch.tensor(cuts, dtype=torch.int32)
        slots = torch.randperm(n, generator=g)[:3].int()
        return (rand(g, rows, ch, t=t), rand(g, rows, 2, 64, t=t), rand(g, rows, 2, t=t),
                rand(g, rows, 2, t=t), rand(g, n, 3, ch, t=t), rand(g, n, 2, 64, 64), off, slots)

    def eager(step):
        mixed, z, b, a, cs, st, off, slots = (x.clone().cuda() for x in step)
        work, out = torch.zeros_like(mixed), torch.zeros_like(z)
        torch.cuda.synchronize()
        mixer(mixed, z, b, a, cs, st, SeqBatch(off, rows, rows, n, slots=slots), work, out)
        block.sync()
        return out[:int(off[-1])], cs, st

    steps = [fresh_step(i, c) for i, c in enumerate([[0, 100, 101, 120], [0, 1, 2, 3],
                                                     [0, 33, 97, 110], [0, 0, 64, 65]])]
    want = [eager(s) for s in steps]
    live = [x.clone().cuda() for x in steps[0]]
    work, out = torch.zeros_like(live[0]), torch.zeros_like(live[1])
    batch = SeqBatch(live[6], rows, rows, n, slots=live[7])
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    block.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=stream):
            mixer(live[0], live[1], live[2], live[3], live[4], live[5], batch, work, out)
    finally:
        block.set_stream(None)
    block.sync()
    big = [400, 33]
    for i, step in enumerate(steps):
        for dst, src in zip(live, step):
            dst.copy_(src)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        block.sync()
        wo, wc, ws = want[i]
        assert torch.equal(out[: wo.shape[0]], wo)
        assert torch.equal(live[4], wc) and torch.equal(live[5], ws)
        run_delta(block, [x * (i + 1) for x in big], 1, 2, 64, 64, t)
    del graph


def test_capture_needs_the_buffers(block):
    """A captured call that would have to allocate is refused and leaves the
    capture whole; after an eager call of its sizes it is taken."""
    from dismoen import MoEBlock
    g = gen("capture")
    with MoEBlock(0) as blk:  # without buffers of other calls
        s = Seqs([70, 30], g, fresh=False)
        q, k, v, a, b, gates = delta_inputs(g, s.rows, 1, 2, 64, 64, torch.bfloat16)
        op = GatedDelta(blk, 1, 2, 64, 64, **gates)
        state, o = rand(g, s.num_slots, 2, 64, 64), torch.zeros_like(v)
        mark = torch.zeros(1, device="cuda")
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        blk.set_stream(stream.cuda_stream)
        with torch.cuda.graph(graph, stream=stream):
            with pytest.raises(DismoenError, match="before the capture"):
                op(q, k, v, a, b, state, s.batch, o)
            mark.add_(1)
        blk.set_stream(None)
        graph.replay()
        torch.cuda.synchronize()
        assert mark.item() == 1 and not o.any()
        start, eager = state.clone(), torch.zeros_like(v)
        torch.cuda.synchronize()
        op(q, k, v, a, b, state, s.batch, eager)
        blk.sync()
        want = state.clone()
        graph2 = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        blk.set_stream(stream.cuda_stream)
        with torch.cuda.graph(graph2, stream=stream):
            op(q, k, v, a, b, state, s.batch, o)
        blk.set_stream(None)
        for _ in range(3):
            state.copy_(start)
            o.zero_()
            torch.cuda.synchronize()
            graph2.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, eager) and torch.equal(state, want)
        blk.sync()
        del graph, graph2


def test_delta_many_chunks(block):
    """More chunks than are worked on at once: the state passes from one part of
    the call to the next in memory."""
    g = gen("parts")
    lens = [20000, 33, 14000]  # 313 + 1 + 219 chunks of 64
    s = Seqs(lens, g, fresh=False)
    q, k, v, a, b, gates = delta_inputs(g, s.rows, 1, 1, 8, 8, torch.float32)
    state, o = rand(g, s.num_slots, 1, 8, 8), torch.zeros_like(v)
    old = state.clone()
    torch.cuda.synchronize()
    op = GatedDelta(block, 1, 1, 8, 8, **gates)
    op(q, k, v, a, b, state, s.batch, o)
    block.sync()
    want, new, largest = R.delta(q, k, v, a, b, old, *s.args, **gates)
    # (a row's roundings fade with the state: those of the last 2000 rows are far
    # more than are left)
    m = float(largest.max())
    live = ~want.isnan()
    R.close(o.cpu()[live], want[live], m * 8 ** -0.5, 64 * 2000)
    R.close(state, new, m, 64 * 2000)


def test_port_block(block, oracle):
    """A whole block: norm, the caller's mixer, residual and norm, MoE section."""
    from dismoen import MoEBlock, PortBlock, synth
    with MoEBlock(0) as blk:
        L = synth.make_layer(**synth.CONFIG_TOY, seed=3)
        blk.upload_layer(0, L)
        g = gen("port")
        h, rows = L.hidden, 9
        x, gi, gp = rand(g, rows, h), 1 + 0.1 * rand(g, h), 1 + 0.1 * rand(g, h)
        w = rand(g, h, h) * h ** -0.5
        port = PortBlock(blk, 0, gi, gp)
        xn, mid, y = (torch.empty_like(x) for _ in range(3))

        def mix(v):
            blk.sync()  # torch's stream is another one
            out = (v @ w).bfloat16()
            torch.cuda.synchronize()
            return out

        torch.cuda.synchronize()
        port(x, mix, xn, mid, y)
        blk.sync()
        _, n1, _ = R.norm(x[:, None], post=False, edge_gamma=gi)
        m = (n1[:, 0].float().cuda() @ w).bfloat16().double().cpu()
        s, n2, _ = R.norm(m[:, None], post=False, residual=x[:, None], edge_gamma=gp)
        # (mix's own rounding to bf16 may fall on the other side)
        assert (mid.cpu().double() - s[:, 0]).abs().max() < 2.0 ** -7 * float(m.abs().max())
        assert (xn.cpu().double() - n2[:, 0]).abs().max() < 2.0 ** -5
        want, ids, _, _ = oracle.moe_layer_q4(L, xn.cpu().numpy(), rows)
        moe = y.cpu().numpy() - mid.cpu().numpy()
        rms = float(np.sqrt(np.mean(want.astype(np.float64) ** 2)))
        # (y - x_mid gives back the sum's own rounding: half a step of values below 8)
        assert np.abs(moe - want).max() <= 1e-3 * rms + 2.0 ** -21
