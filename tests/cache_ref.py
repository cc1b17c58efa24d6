"""The 4-bit cache and attention over it from their definitions, in 64 bits on the CPU."""
import numpy as np
import torch

LEVELS = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def held(x):
    """What the cache holds of rows [..., dim]."""
    x = x.double().cpu().unflatten(-1, (-1, 32))
    most = x.abs().amax(-1, keepdim=True)
    unit = torch.full_like(most, 2.0 ** -120)
    for p in range(-119, 126):
        unit = torch.where(most > 7 * unit, torch.full_like(unit, 2.0 ** p), unit)
    y = (x / unit).abs().unsqueeze(-1)
    off = (y - LEVELS).abs()
    # ties to the even code: its distance counts a little less
    off = off - torch.where(torch.arange(8) % 2 == 0, 1e-9, 0.0)
    v = LEVELS[off.argmin(-1)] * unit * torch.where(x < 0, -1.0, 1.0)
    return torch.where(most.isfinite(), v, torch.full_like(v, float("nan"))).flatten(-2)


def attend(q, k, v, past, scale, gate=None):
    """(o, size) of rows q [n][heads][dim] at positions past + t over k, v [past + n]
    [kv_heads][dim]; size: sum of p |v| times the gate, what the roundings of p and of the
    sums count against, and the largest |z| of a row in front of it."""
    n, heads, d = q.shape
    rep = heads // k.shape[1]
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    o, size = torch.empty_like(q), torch.empty_like(q)
    for h in range(heads):
        for t in range(n):
            kk, vv = k[:past + t + 1, h // rep], v[:past + t + 1, h // rep]
            z = scale * (kk @ q[t, h])
            p = (z - z.max()).exp()
            p = p / p.sum()
            o[t, h] = p @ vv
            # an error of a score is its terms' roundings
            terms = scale * (kk.abs() @ q[t, h].abs()).max()
            size[t, h] = (p @ vv.abs()) * (1 + terms)
    if gate is not None:
        g = torch.sigmoid(gate.double().cpu())
        o, size = o * g, size * g
    return o, size


def i32(x, device="cuda"):
    return torch.as_tensor(np.asarray(x, np.int32)).to(device)
