"""The bounds that the delta rule's kernels are held to (delta_forms), without a
GPU: the chunked form in fp32 keeps them, one with fewer parts does not."""
import pytest
import torch

import delta_forms as D

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def inputs(t, hk, hv, dk, dv, n):
    torch.manual_seed(n * 1000 + dk)
    x = torch.randn(n, 2 * hk * dk + hv * dv)
    x = (x * torch.sigmoid(x)).to(t)
    q, k = (x[:, i * hk * dk:(i + 1) * hk * dk].unflatten(1, (hk, dk)) for i in (0, 1))
    v = x[:, 2 * hk * dk:].unflatten(1, (hv, dv))
    g, beta = D.gates(torch.randn(n, hv).to(t), torch.randn(n, hv).to(t), torch.randn(hv),
                      torch.randn(hv) - 2)
    return q, k, v, g, beta, torch.randn(hv, dk, dv) * 0.3


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(2, 4, 128, 128, 150), (1, 2, 64, 24, 300), (1, 2, 256, 40, 70),
                                   (1, 1, 8, 8, 130)], ids=str)
def test_bounds_tell_parts_apart(shape, t):
    ins = inputs(t, *shape)

    def worst(parts, out_parts):
        o, s = D.chunked(*ins, parts, out_parts)
        return D.check(o.to(t), s, *ins)

    assert max(worst(3, 3)) <= 1
    assert worst(2, 3)[1] > 2
    if t is torch.float32:
        assert worst(3, 2)[0] > 2


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("dk", [64, 128])
def test_cancelling_outputs_tell_parts_apart(dk, t):
    ins, want, tol = D.cancelling(t, dk, 40)
    for out_parts, holds in ((3, True), (2, False)):
        o, _ = D.chunked(*ins, 3, out_parts, eps=0.0, scale=1.0)
        off = (o.to(t).double() - want).abs() / tol
        for rows in (slice(2, 64), slice(64, None)):
            assert (float(off[rows].max()) <= 1) == holds
