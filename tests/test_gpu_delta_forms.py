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
