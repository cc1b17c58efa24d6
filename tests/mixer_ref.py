"""The token mixer's operators from their definitions, in 64 bits on the CPU,
and how far a result rounded to a type may be from them."""
import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def close(got, want, scale, steps):
    """|got - want| within one rounding to got's type of the value and `steps`
    roundings of 2^-24 of quantities as large as `scale` (which broadcasts)."""
    got, want = got.detach().cpu(), want.cpu()
    tol = want.abs() * HALF_STEP[got.dtype] * (1 + 2.0 ** -10) + SMALLEST[got.dtype]
    tol = tol + steps * 2.0 ** -24 * scale
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (
        f"{int(bad.sum())} of {bad.numel()} off, most "
        f"{float(((got.double() - want).abs() / tol).max()):.3g} times the tolerance")


def seqs_of(offsets, slots, fresh, num_slots):
    for i in range(len(offsets) - 1):
        b, e = int(offsets[i]), int(offsets[i + 1])
        slot = i if slots is None else int(slots[i])
        if slot >= 0 and e > b:
            yield i, b, e, slot, bool(fresh is not None and int(fresh[i]))


def conv(x, weight, bias, state, offsets, slots=None, fresh=None, silu=True):
    """(y, state, size): y rows of no sequence are NaN; size bounds what a row sums."""
    x, w = x.double().cpu(), weight.double().cpu()
    state = state.double().cpu().clone()
    y = torch.full_like(x, float("nan"))
    size = torch.zeros_like(x)
    width = w.shape[1]
    for _, b, e, slot, new in seqs_of(offsets, slots, fresh, state.shape[0]):
        line = torch.cat([state[slot] * (0 if new else 1), x[b:e]])
        for t in range(e - b):
            terms = line[t:t + width].T * w
            z = terms.sum(1) + (0 if bias is None else bias.double().cpu())
            y[b + t] = z * torch.sigmoid(z) if silu else z
            size[b + t] = terms.abs().sum(1) + (0 if bias is None else bias.double().cpu().abs())
        state[slot] = line[e - b:]
    return y, state, size


def norm(x, gamma=None, post=True, gate=None, act=None, residual=None, scale=1.0,
         edge_gamma=None, eps=1e-6):
    """(stream, y, size of stream's terms)"""
    u = x.double().cpu()
    if post:
        u = u / (u.square().mean(-1, keepdim=True) + eps).sqrt()
        u = u if gamma is None else u * gamma.double().cpu()
    if act:
        z = gate.double().cpu()
        u = u * (z * torch.sigmoid(z) if act == "silu" else torch.sigmoid(z))
    u = u * (scale if isinstance(scale, float) else scale.double().cpu())
    size = u.abs()
    if residual is not None:
        u = u + residual.double().cpu()
        size = size + residual.double().cpu().abs()
    y = u / (u.square().mean(-1, keepdim=True) + eps).sqrt()
    return u, (y if edge_gamma is None else y * edge_gamma.double().cpu()), size


def delta(q, k, v, a, b, state, offsets, slots=None, fresh=None, a_log=None, dt_bias=None,
          qk_norm=True, eps=1e-6, scale=None):
    """(o, state, largest): o rows of no sequence are NaN; largest [slots][heads]:
    the largest norm that a column of the state, or element of v, had on the way."""
    q, k, v, a, b = (t.double().cpu() for t in (q, k, v, a, b))
    rep, dk = v.shape[1] // q.shape[1], q.shape[2]
    scale = dk ** -0.5 if scale is None else scale
    state = state.double().cpu().clone()
    o = torch.full_like(v, float("nan"))
    if a_log is not None:
        g = a if dt_bias is None else a + dt_bias.double().cpu()
        g = -a_log.double().cpu().exp() * torch.where(g > 40, g, g.clamp(max=40).exp().log1p())
        beta = torch.sigmoid(b)
    else:
        g, beta = a, b
    largest = state.square().sum(2).sqrt().amax(2)
    for _, at, end, slot, new in seqs_of(offsets, slots, fresh, state.shape[0]):
        s = state[slot] * 0 if new else state[slot]
        for t in range(at, end):
            kt, qt = k[t].repeat_interleave(rep, 0), q[t].repeat_interleave(rep, 0)
            if qk_norm:
                kt = kt / (kt.square().sum(1, keepdim=True) + eps).sqrt()
                qt = qt / (qt.square().sum(1, keepdim=True) + eps).sqrt()
            s = g[t].exp()[:, None, None] * s
            u = beta[t][:, None] * (v[t] - (kt[:, :, None] * s).sum(1))
            s = s + kt[:, :, None] * u[:, None, :]
            o[t] = scale * (qt[:, :, None] * s).sum(1)
            largest[slot] = torch.maximum(largest[slot], torch.maximum(
                s.square().sum(1).sqrt().amax(1), v[t].abs().amax(1)))
        state[slot] = s
    return o, state, largest


def bf16_bits(t):
    return t.view(torch.int16).numpy().view(np.uint16)
