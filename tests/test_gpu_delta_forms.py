"""Every form of the chunked delta rule on the GPU (row type, key dimension, one or
two column tiles a workgroup, one or two value heads a key head), held to the bounds
of delta_forms; and a sequence's bits alone, where it takes one column tile,
against those in a call that takes two."""
import pytest
import torch

import delta_forms as D
from dismoen import GatedDelta, SeqBatch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def i32(*v):
    return torch.tensor(v, dtype=torch.int32).cuda()


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("k_dim,v_dim", [(64, 32), (64, 40), (128, 72), (256, 16)])
def test_outputs_that_cancel(block, k_dim, v_dim, t):
    (q, k, v, g, beta, state), want, tol = D.cancelling(t, k_dim, v_dim)
    n = q.shape[0]
    op = GatedDelta(block, 1, v.shape[1], k_dim, v_dim, eps=0.0, scale=1.0)
    o, s = torch.zeros_like(v).cuda(), state[None].cuda()
    ins = [x.cuda() for x in (q, k, v, g.float(), beta.float())]
    batch = SeqBatch(i32(0, n), n, n, 1)
    torch.cuda.synchronize()
    op(*ins, s, batch, o)
    block.sync()
    off = (o.cpu().double() - want).abs() / tol
    assert float(off.max()) <= 1, [float(off[:64].max()), float(off[64:].max())]


# Sequences of more than 16 rows in chunks, of whole chunks, one row and none.  The
# chunked form takes two column tiles of 16 a workgroup where those of all sequences
# that could be longer than 16 rows are more than 256: here 6 times the value heads
# times the tiles of v_dim; of one sequence alone they are fewer.
LENS = [130, 1, 64, 40, 0, 17]
SHAPES = [(64, 2, 6, 136), (56, 4, 4, 200), (128, 4, 8, 136), (120, 8, 8, 136), (72, 4, 16, 40),
          (256, 2, 6, 136), (136, 4, 4, 200), (248, 4, 16, 40)]


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("k_dim,hk,hv,v_dim", SHAPES)
def test_forms(block, k_dim, hk, hv, v_dim, t):
    tiles = hv * ((v_dim + 15) // 16)
    assert len(LENS) * tiles > 256 >= tiles
    g = torch.Generator().manual_seed(k_dim + v_dim)
    n, rows = len(LENS), sum(LENS)
    x = torch.randn((rows, 2 * hk * k_dim + hv * v_dim), generator=g)
    x = (x * torch.sigmoid(x)).to(t)
    q, k = (x[:, i * hk * k_dim:(i + 1) * hk * k_dim].unflatten(1, (hk, k_dim)) for i in (0, 1))
    v = x[:, 2 * hk * k_dim:].unflatten(1, (hv, v_dim))
    a, b = (torch.randn((rows, hv), generator=g).to(t) for _ in range(2))
    a_log, dt_bias = torch.randn(hv, generator=g), torch.randn(hv, generator=g) - 2
    start = torch.randn((n, hv, k_dim, v_dim), generator=g) * 0.3
    off = [sum(LENS[:i]) for i in range(n + 1)]
    op = GatedDelta(block, hk, hv, k_dim, v_dim, a_log=a_log.cuda(), dt_bias=dt_bias.cuda())
    x = x.cuda()
    dq, dk = (x[:, i * hk * k_dim:(i + 1) * hk * k_dim].unflatten(1, (hk, k_dim)) for i in (0, 1))
    dv = x[:, 2 * hk * k_dim:].unflatten(1, (hv, v_dim))
    ins = (dq, dk, dv, a.cuda(), b.cuda())
    o, state = torch.zeros((rows, hv, v_dim), dtype=t, device="cuda"), start.cuda()
    torch.cuda.synchronize()
    op(*ins, state, SeqBatch(i32(*off), rows, max(LENS), n), o)
    block.sync()
    log_decay, beta = D.gates(a, b, a_log, dt_bias)
    for i, length in enumerate(LENS):
        at = slice(off[i], off[i + 1])
        if not length:
            assert torch.equal(state[i].cpu(), start[i])
            continue
        worst = D.check(o[at], state[i], q[at], k[at], v[at], log_decay[at], beta[at], start[i])
        assert max(worst) <= 1, (length, worst)
        alone, one = torch.zeros_like(o[at]), start[i:i + 1].cuda()
        torch.cuda.synchronize()
        op(*(y[at] for y in ins), one, SeqBatch(i32(0, length), length, length, 1), alone)
        block.sync()
        assert torch.equal(alone, o[at]) and torch.equal(one[0], state[i]), length


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES)
def test_a_prompt_among_single_tokens(block, t):
    """The sequences of one row outnumber the chunked ones by far, on both sides of them."""
    lens = [1] * 70 + [150] + [1] * 40 + [0, 70] + [1] * 9
    hk, hv, dk, dv, n, rows = 2, 4, 64, 64, len(lens), sum(lens)
    g = torch.Generator().manual_seed(9)
    q, k = (torch.randn((rows, hk, dk), generator=g).to(t) for _ in range(2))
    v = torch.randn((rows, hv, dv), generator=g).to(t)
    a, b = -torch.rand((rows, hv), generator=g), torch.rand((rows, hv), generator=g)
    start = torch.randn((n, hv, dk, dv), generator=g) * 0.3
    slots = torch.randperm(n, generator=g).int()
    off = [sum(lens[:i]) for i in range(n + 1)]
    o, state = torch.zeros((rows, hv, dv), dtype=t, device="cuda"), start.cuda()
    ins = [x.cuda() for x in (q, k, v, a, b)]
    batch = SeqBatch(i32(*off), rows, max(lens), n, slots=slots.cuda())
    torch.cuda.synchronize()
    GatedDelta(block, hk, hv, dk, dv)(*ins, state, batch, o)
    block.sync()
    for i in range(n):
        at, slot = slice(off[i], off[i + 1]), int(slots[i])
        if not lens[i]:
            assert torch.equal(state[slot].cpu(), start[slot])
            continue
        worst = D.check(o[at], state[slot], q[at], k[at], v[at], a[at].double(), b[at].double(),
                        start[slot])
        assert max(worst) <= 1, (i, worst)
