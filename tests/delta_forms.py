"""The gated delta rule in fp32, on the CPU: row by row, and 64 rows at a time
with the factors of its products in a given number of bf16 parts.  What the
first is off from 64 bits bounds what a kernel that computes in fp32 may be off;
the second, with fewer parts than fp32 holds, is what has to exceed the bound.

Bounds.  A row by row loop in fp32 makes some 2 (k_dim + 8) roundings of 2^-24 per
row, most of them in its sums; the chunked form sums as much over k_dim, twice 64
products more in T R and K^T U, and drops products of parts below 2^-26 of a
factor: up to twice as many roundings per row for dimensions from 64 on, more for
smaller ones, and its sums in another order.  Roundings add up like random numbers in
both, so the chunked state may be FACTOR = 8 times as far off in the 2-norm of a
head; an element is within 6 times its head's root mean square in all but one of
10^9, so an output may be 6 FACTOR times the loop's root mean square off, over the
rows of 64 around it, and half a step of its type.  The floor under the loop's own
error is half a rounding of the value: 2^-25 of the 2-norm."""
import torch

FACTOR = 8
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def gates(a, b, a_log, dt_bias):
    """(log decay, beta) of raw or final gates, in 64 bits."""
    a, b = a.double().cpu(), b.double().cpu()
    if a_log is None:
        return a, b
    x = a if dt_bias is None else a + dt_bias.double().cpu()
    g = -a_log.double().cpu().exp() * torch.where(x > 40, x, x.clamp(max=40).exp().log1p())
    return g, torch.sigmoid(b)


def heads(q, k, v, eps, scale):
    """q, k of every value head, normalised, q scaled: [heads][rows][dim]; v as well."""
    rep = v.shape[1] // q.shape[1]
    q, k = (x.repeat_interleave(rep, 1).transpose(0, 1) for x in (q, k))
    q = q / (q.square().sum(-1, keepdim=True) + eps).sqrt() * scale
    return q, k / (k.square().sum(-1, keepdim=True) + eps).sqrt(), v.transpose(0, 1)


def loop(q, k, v, g, beta, state, dtype, eps=1e-6, scale=None):
    """One sequence row by row: (o [rows][heads][v_dim], state) in dtype."""
    scale = q.shape[2] ** -0.5 if scale is None else scale
    q, k, v = heads(*(x.cpu().to(dtype) for x in (q, k, v)), eps, scale)
    grow, beta = g.to(dtype).exp(), beta.to(dtype)
    s = state.cpu().to(dtype)
    o = torch.empty_like(v)
    for t in range(v.shape[1]):
        s = s * grow[t][:, None, None]
        u = beta[t][:, None] * (v[:, t] - (k[:, t, None] @ s)[:, 0])
        s = s + k[:, t, :, None] * u[:, None]
        o[:, t] = (q[:, t, None] @ s)[:, 0]
    return o.transpose(0, 1), s


def split(x, n):
    """x as n parts of 8 bits."""
    parts = []
    for _ in range(n):
        p = x.float().bfloat16().double()
        parts.append(p)
        x = x - p
    return parts


def product(a, b, n):
    """a b of factors in n parts, those products that i + j < n, rounded to fp32."""
    pa, pb = split(a, n), split(b, n)
    return sum(pa[i] @ pb[j] for i in range(n) for j in range(n - i)).float().double()


def chunked(q, k, v, g, beta, state, parts, out_parts, eps=1e-6, scale=None):
    """One sequence 64 rows at a time, what reaches the state in `parts` parts and
    what reaches the outputs alone in `out_parts`: (o, state) in fp32 values."""
    scale = q.shape[2] ** -0.5 if scale is None else scale
    q, k, v = heads(*(x.cpu().double() for x in (q, k, v)), eps, scale)
    s, os = state.cpu().double(), []
    for at in range(0, v.shape[1], 64):
        qc, kc, vc = (x[:, at:at + 64] for x in (q, k, v))
        since = g[at:at + 64].T.cumsum(1)
        b = beta[at:at + 64].T[:, :, None]
        gone = (since[:, :, None] - since[:, None]).tril().exp().tril()
        n = vc.shape[1]
        low = (b * (kc @ kc.transpose(1, 2)) * gone).tril(-1).float().double()
        t = (torch.linalg.inv(torch.eye(n, dtype=torch.double) + low) * b.transpose(1, 2))
        grow, rest = since.exp()[:, :, None], (since[:, -1:] - since).exp()[:, :, None]
        r = (vc - (grow * product(kc, s, parts)).float().double()).float().double()
        u = product(t.float().double(), r, parts)
        qk = ((qc @ kc.transpose(1, 2)) * gone).float().double()
        os.append((grow * product(qc, s, out_parts) + product(qk, u, out_parts)).float())
        s = (grow[:, -1:] * s + product(kc.transpose(1, 2), rest * u, parts)).float().double()
    return torch.cat(os, 1).transpose(0, 1), s.float()


def check(o, state, q, k, v, g, beta, start, eps=1e-6, scale=None):
    """One sequence's outputs and state, given as they came, against 64 bits: the
    worst ratio to the bound of each; at most 1 where they hold."""
    o64, s64 = loop(q, k, v, g, beta, start, torch.double, eps, scale)
    o32, s32 = loop(q, k, v, g, beta, start, torch.float, eps, scale)
    o, state = o.detach().cpu(), state.detach().cpu()

    def size(x):  # 2-norm of a head's state
        return x.double().square().sum((1, 2)).sqrt()

    floor = 2.0 ** -25
    bound = FACTOR * torch.maximum(size(s32.double() - s64), floor * size(s64)) + 2.0 ** -149
    in_state = float((size(state.double() - s64) / bound).max())
    worst = 0.0
    for at in range(0, o.shape[0], 64):  # the root mean square of these rows, per head
        want, off = o64[at:at + 64], o32[at:at + 64].double() - o64[at:at + 64]
        rms = torch.maximum(off.square().mean((0, 2)).sqrt(),
                            floor * want.square().mean((0, 2)).sqrt())[:, None]
        tol = want.abs() * HALF_STEP[o.dtype] * (1 + 2.0 ** -10) + SMALLEST[o.dtype]
        tol = tol + 6 * FACTOR * rms
        worst = max(worst, float(((o[at:at + 64].double() - want).abs() / tol).max()))
    return worst, in_state


def cancelling(t, k_dim, v_dim, heads=2, rows=80):
    """One sequence whose outputs nearly cancel, from a state of zeros, without
    decay: (inputs of the other functions, the outputs in 64 bits, what they may be
    off).  Keys are unit vectors, two of a kind nowhere, so row t writes beta v at
    its own dimension and nothing else there; the rows come in pairs of -v and v
    whose betas are 2^-14 apart, and queries ask for the sum of a pair: within the
    first 64 rows through the query-key matrix, behind them through the state.
    Off by 24 roundings of 2^-24 of beta v at most (each u of the pair: the sum of
    its product's six parts, 5, and what three parts leave, 1; the sum of the six
    parts of what reads both, 6, and three leave, 1; the rows' factors, 3; one to
    spare), and by half a step of the result's type."""
    g = torch.Generator().manual_seed(k_dim)
    k = torch.zeros(rows, 1, k_dim)
    k[torch.arange(64), 0, torch.arange(64)] = 1
    v = torch.randn(rows, heads, v_dim, generator=g).to(t)
    v[1::2] = -v[::2]
    beta = 0.5 + 0.4 * torch.rand(rows, heads, generator=g)
    beta[1::2] = beta[::2] * (1 + 2.0 ** -14)
    beta[64:] = 0
    k[64:, 0, 0] = 1  # (written with nothing)
    pair = torch.tensor([int(torch.randint(min(i + 1, 64) // 2, (), generator=g)) if i else 0
                         for i in range(rows)])
    q = torch.zeros(rows, 1, k_dim)
    q[torch.arange(rows), 0, 2 * pair] = 1
    q[torch.arange(rows), 0, 2 * pair + 1] = 1
    beta = beta.double()  # (fp32 values)
    u = beta[:, :, None] * v.double()
    # (keys that are not normalised: eps 0 and unit vectors; queries of norm sqrt 2)
    root = 2.0 ** -0.5
    want = (u[2 * pair] + torch.where((2 * pair + 1 <= torch.arange(rows))[:, None, None],
                                      u[2 * pair + 1], 0.0)) * root
    tol = want.abs() * HALF_STEP[t] * (1 + 2.0 ** -10) + SMALLEST[t]
    tol = tol + 24 * 2.0 ** -24 * root * u[2 * pair].abs()
    state = torch.zeros(heads, k_dim, v_dim)
    return (q.to(t), k.to(t), v, torch.zeros(rows, heads).double(), beta, state), want, tol
