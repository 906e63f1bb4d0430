"""Some rows of a call with shaped scores, and the weights of some keys, in 64 bits, where all of them would take minutes (scored_reference has the
definition and where the tolerances come from; they are the same here)."""
import math

import torch


def scores_of(c, b, h, idx, keys):
    """As Case.scores, of the new tokens idx and the keys `keys` of a sequence: (visible, scores, how far off in units of their exponents)."""
    n, L, g = c.news[b], c.lens[b], h // (c.heads // c.kv_heads)
    place = torch.tensor([-1 if c.row(b, int(j)) is None else c.row(b, int(j)) for j in keys])
    k = torch.where((place >= 0)[:, None], c.k[place.clamp(min=0), g, keys % c.page].double(), 0.0)
    p, j = (L - n + idx)[:, None], keys[None, :]
    near = torch.ones(len(idx), len(keys), dtype=torch.bool)
    if c.window:
        near &= j > p - c.window
    if c.first is not None:
        near &= j >= torch.tensor(c.first)[int(c.starts[b]) + idx][:, None]
    if c.sinks:
        near |= j < c.sinks
    ok = near & (j <= p) if c.causal else near
    if c.prefix is not None:
        ok |= j < c.prefix[b]
    ok &= (place >= 0)[None, :]
    q = c.q[int(c.starts[b]) + idx, h].double()
    x = q @ k.T * c.scale
    off = (c.dim + 4) * (q.abs() @ k.abs().T * c.scale) + 4
    if c.cap:
        x = c.cap * torch.tanh(x / c.cap)
        off = off + 8 * c.cap
    if c.slopes is not None:
        s, far = torch.tensor(c.slopes[h], dtype=torch.float32).double(), (p - j).abs().double()
        x = x - s * far
        off = off + 4 * s.abs() * far
    off = off + 2 * x.abs()
    return ok, torch.where(ok, x, -math.inf), torch.where(ok, 2 * off * 2.0 ** -24, 0.0)


def rows(c, b, h, idx):
    """(out, lse, tolerances of both) of new tokens idx of a sequence, query head h."""
    keys = torch.arange(c.lens[b])
    g = h // (c.heads // c.kv_heads)
    ok, s, off = scores_of(c, b, h, idx, keys)
    v, _ = c.rows(c.v, b, g)
    u = 2.0 ** -8 if c.dtype == "bf16" else 2.0 ** -11
    z = torch.logsumexp(s, dim=1)
    p = torch.where(ok, torch.exp(s - torch.where(z == -math.inf, 0.0, z)[:, None]), 0.0)
    o = torch.stack([(p[i][ok[i]][:, None] * v[ok[i]]).sum(dim=0) for i in range(len(idx))])
    size = v.abs().nan_to_num(0, 0, 0)
    sums = (p * off).sum(dim=1) + (ok.sum(dim=1) + 8) * 2.0 ** -23
    tol = u * o.abs().nan_to_num(0, 0, 0) + ((p * (u + off)) @ size + sums[:, None] * (p @ size)) * (1 + 2 * u)
    if c.dtype == "fp16":
        tol += 2.0 ** -25 * (1 + ok.double() @ size)
    return o, z, tol, sums + 2.0 ** -22 * (1 + z.abs().nan_to_num(0, 0, 0))


def weights(c, b, g, keys, lse):
    """(what the keys `keys` of a sequence drew from the query heads of KV head g, how far off), for the lse that the call is given.  Each weight below
    2^-126, the least normal number of 32 bits, is 0: a sum is off by as many of them as it has terms at most."""
    group, idx = c.heads // c.kv_heads, torch.arange(c.news[b])
    t = slice(int(c.starts[b]), int(c.starts[b + 1]))
    w, err = torch.zeros(len(keys), dtype=torch.float64), torch.zeros(len(keys), dtype=torch.float64)
    for h in range(g * group, (g + 1) * group):
        z = lse[h, t].double()
        ok, s, off = scores_of(c, b, h, idx, keys)
        use = ok & (z != -math.inf)[:, None]
        p = torch.where(use, torch.exp(s - z[:, None]), 0.0)
        e = off + (4 * z.abs().nan_to_num(0, 0, 0)[:, None] + 8 + use.sum(dim=0)[None, :] * group) * 2.0 ** -24
        w += p.sum(dim=0)
        err += torch.where(use, 2 * e * p, 0.0).sum(dim=0)
    return w, err + group * c.news[b] * 2.0 ** -126
