"""Attention over a paged cache with capped, sloped and masked scores, and the weights that it gives, in 64 bits, row by row; and how far 32-bit
scores and 16-bit roundings may carry a kernel from them.

A score's exponent is off by: the product's d terms (d + 4 half steps of the sum of their sizes); a cap: the argument of the exponential, the
exponential, the reciprocal and the last sum, together less than 2^-21 of the cap, on top of the product's error, which a cap makes no larger; a slope: its
own rounding to units of log2, the product's and the sum's, 2^-24 each of slope times distance; and the difference from the reference. Twice that, for the
reference is such a score itself.  Probabilities are rounded to the storage type, O in the end."""
import math

import torch

import paged_reference as ref


class Case(ref.Case):
    """ref.Case with scoring: cap; slopes, a number for every head; prefix, a number for every sequence; first, a number for every token."""

    def __init__(self, cap=0.0, slopes=None, prefix=None, first=None, **more):
        super().__init__(**more)
        self.cap, self.slopes, self.prefix, self.first = cap, slopes, prefix, first

    def given(self):
        """(slopes, prefix_lens, first_keys) on the device."""
        made = lambda x, t: None if x is None else torch.tensor(x, dtype=t).cuda()   # noqa: E731
        return made(self.slopes, torch.float32), made(self.prefix, torch.int32), made(self.first, torch.int32)

    def sight(self, b, there):
        """[new tokens, keys] visible, [new tokens, keys] distances."""
        n, L = self.news[b], self.lens[b]
        p, j = (L - n + torch.arange(n))[:, None], torch.arange(L)[None, :]
        ok = j <= p if self.causal else torch.ones(n, L, dtype=torch.bool)
        near = torch.ones(n, L, dtype=torch.bool)
        if self.window:
            near &= j > p - self.window
        if self.first is not None:
            near &= j >= torch.tensor(self.first[int(self.starts[b]):int(self.starts[b + 1])])[:, None]
        if self.sinks:
            near |= j < self.sinks
        ok = ok & near
        if self.prefix is not None:
            ok = ok | (j < self.prefix[b])
        return ok & there[None, :], (p - j).abs()

    def scores(self, b, h, k, there):
        """(visible, scores with -inf where hidden, how far a visible one's exponent may be off) of a query head of a sequence."""
        t = slice(int(self.starts[b]), int(self.starts[b + 1]))
        ok, far = self.sight(b, there)
        q, d = self.q[t, h].double(), self.dim
        k = torch.where(there[:, None], k, 0.0)
        x = q @ k.T * self.scale
        off = (d + 4) * (q.abs() @ k.abs().T * self.scale) + 4
        if self.cap:
            x = self.cap * torch.tanh(x / self.cap)
            off = off + 8 * self.cap
        if self.slopes is not None:
            s = torch.tensor(self.slopes[h], dtype=torch.float32).double()
            x = x - s * far
            off = off + 4 * s.abs() * far
        off = off + 2 * x.abs()
        return ok, torch.where(ok, x, -math.inf), torch.where(ok, 2 * off * 2.0 ** -24, 0.0)


def attend(c):
    """As ref.attend."""
    T, H, d = c.tokens, c.heads, c.dim
    out, tol = torch.zeros(T, H, d, dtype=torch.float64), torch.zeros(T, H, d, dtype=torch.float64)
    lse, tol_lse = torch.full((H, T), -math.inf, dtype=torch.float64), torch.zeros(H, T, dtype=torch.float64)
    u = 2.0 ** -8 if c.dtype == "bf16" else 2.0 ** -11
    for b in range(len(c.lens)):
        if not c.news[b] or not c.lens[b]:
            continue
        t = slice(int(c.starts[b]), int(c.starts[b + 1]))
        for h in range(H):
            g = h // (H // c.kv_heads)
            (k, there), (v, _) = c.rows(c.k, b, g), c.rows(c.v, b, g)
            ok, s, off = c.scores(b, h, k, there)
            z = torch.logsumexp(s, dim=1)
            p = torch.where(ok, torch.exp(s - torch.where(z == -math.inf, 0.0, z)[:, None]), 0.0)
            some = ok.any(dim=0)   # (keys that no row sees may hold anything)
            o = p @ torch.where(some[:, None], v, 0.0) if torch.isfinite(v[some]).all() else torch.stack(
                [(p[i][ok[i]][:, None] * v[ok[i]]).sum(dim=0) for i in range(p.shape[0])])
            size = torch.where(some[:, None], v, 0.0).abs().nan_to_num(0, 0, 0)
            sums = (p * off).sum(dim=1) + (ok.sum(dim=1) + 8) * 2.0 ** -23   # of the weights' sum
            out[t, h], lse[h, t] = o, z
            tol[t, h] = u * o.abs().nan_to_num(0, 0, 0) + ((p * (u + off)) @ size + sums[:, None] * (p @ size)) * (1 + 2 * u)
            if c.dtype == "fp16":
                tol[t, h] += 2.0 ** -25 * (1 + ok.double() @ size)
            tol_lse[h, t] = sums + 2.0 ** -22 * (1 + z.abs().nan_to_num(0, 0, 0))
    return out, lse, tol, tol_lse


def weights(c, lse):
    """As ref.weights."""
    scores = torch.zeros(c.pages, c.kv_heads, c.page, dtype=torch.float64)
    tol = torch.zeros_like(scores)
    group = c.heads // c.kv_heads
    for b in range(len(c.lens)):
        if not c.news[b] or not c.lens[b]:
            continue
        t = slice(int(c.starts[b]), int(c.starts[b + 1]))
        for g in range(c.kv_heads):
            k, there = c.rows(c.k, b, g)
            w, err = torch.zeros(c.lens[b], dtype=torch.float64), torch.zeros(c.lens[b], dtype=torch.float64)
            for h in range(g * group, (g + 1) * group):
                z = lse[h, t].double()
                ok, s, off = c.scores(b, h, k, there)
                use = ok & (z != -math.inf)[:, None]
                p = torch.where(use, torch.exp(s - z[:, None]), 0.0)
                e = off + (4 * z.abs().nan_to_num(0, 0, 0)[:, None] + 8 + use.sum(dim=0)[None, :] * group) * 2.0 ** -24
                w += p.sum(dim=0)
                err += torch.where(use, 2 * e * p, 0.0).sum(dim=0)
            for j in range(c.lens[b]):
                page = c.row(b, j)
                if page is not None:
                    scores[page, g, j % c.page] = w[j]
                    tol[page, g, j % c.page] = err[j] + 2.0 ** -126
    return scores, tol
