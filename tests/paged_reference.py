"""The paged cache's operators in 64 bits, and how far 32-bit sums and 16-bit roundings may carry a kernel from them."""
import math

import torch

TORCH = {"fp16": torch.float16, "bf16": torch.bfloat16}


class Case:
    """A ragged batch over a pool of pages, made on the CPU from a seed.  Places that no sequence owns hold `spare` in every row."""

    def __init__(self, dtype="bf16", dim=128, heads=4, kv_heads=2, page=16, lens=(), news=(), window=0, sinks=0, causal=True, seed=0,
                 spare=float("nan"), sigma=1.0, extra_rows=0, extra_pages=2):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.dim, self.heads, self.kv_heads, self.page = dtype, dim, heads, kv_heads, page
        self.lens, self.news, self.window, self.sinks, self.causal = list(lens), list(news), window, sinks, causal
        need = [-(-max(0, n) // page) for n in lens]
        self.pages = sum(need) + extra_pages
        self.table = torch.full((len(lens), max(need + [1]) + 1), -1, dtype=torch.int32)
        order = torch.randperm(self.pages, generator=g)
        at = 0
        shape = (self.pages, kv_heads, page, dim)
        self.k, self.v = torch.full(shape, spare).to(TORCH[dtype]), torch.full(shape, spare).to(TORCH[dtype])
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n].to(torch.int32)
            at += n
            for j in range(n):
                rows = min(page, lens[b] - j * page)
                p = int(self.table[b, j])
                self.k[p, :, :rows] = (sigma * torch.randn(kv_heads, rows, dim, generator=g)).to(TORCH[dtype])
                self.v[p, :, :rows] = torch.randn(kv_heads, rows, dim, generator=g).to(TORCH[dtype])
        self.starts = torch.tensor([sum(self.news[:b]) for b in range(len(news) + 1)], dtype=torch.int32)
        self.tokens = int(self.starts[-1]) + extra_rows
        self.q = (sigma * torch.randn(self.tokens, heads, dim, generator=g)).to(TORCH[dtype])
        self.scale = 1 / math.sqrt(dim)

    def kv_lens(self):
        return torch.tensor(self.lens, dtype=torch.int32)

    def row(self, b, j):
        """Page of token j, or None."""
        p = int(self.table[b, j // self.page]) if j // self.page < self.table.shape[1] else -1
        return p if 0 <= p < self.pages else None

    def rows(self, cache, b, h):
        """[L, ...] rows of a head, 0 where the page is not there, and which are."""
        n = self.lens[b]
        at = torch.tensor([-1 if self.row(b, j) is None else self.row(b, j) for j in range(n)], dtype=torch.long)
        there = at >= 0
        x = cache[at.clamp(min=0), h, torch.arange(n) % self.page]
        x = torch.where(there.reshape([-1] + [1] * (x.dim() - 1)), x.double(), 0.0)
        return x, there

    def seen(self, b, there):
        n, L = self.news[b], self.lens[b]
        p = (L - n + torch.arange(n))[:, None]
        j = torch.arange(L)[None, :]
        ok = there[None, :].expand(n, L).clone()
        if self.causal:
            ok &= j <= p
        if self.window:
            ok &= (j > p - self.window) | (j < self.sinks)
        return ok


def attend(c):
    """(out, lse, how far out may be off, how far lse may be off), in float64; NaN rows of q, K and V spread as the formula says."""
    T, H, d = c.tokens, c.heads, c.dim
    out, tol = torch.zeros(T, H, d, dtype=torch.float64), torch.zeros(T, H, d, dtype=torch.float64)
    lse, tol_lse = torch.full((H, T), -math.inf, dtype=torch.float64), torch.zeros(H, T, dtype=torch.float64)
    u = 2.0 ** -8 if c.dtype == "bf16" else 2.0 ** -11   # half a step of the storage type, relative
    for b in range(len(c.lens)):
        if not c.news[b] or not c.lens[b]:
            continue
        t = slice(int(c.starts[b]), int(c.starts[b + 1]))
        for h in range(H):
            g = h // (H // c.kv_heads)
            k, there = c.rows(c.k, b, g)
            v, _ = c.rows(c.v, b, g)
            ok = c.seen(b, there)
            q = c.q[t, h].double()
            s = torch.where(ok, q @ torch.where(there[:, None], k, 0.0).T * c.scale, -math.inf)
            top = s.amax(dim=1)
            z = torch.logsumexp(s, dim=1)
            p = torch.where(ok, torch.exp(s - torch.where(z == -math.inf, 0.0, z)[:, None]), 0.0)
            # row by row where a value is not finite: a hidden key contributes nothing, whatever its V holds
            if torch.isfinite(v).all():
                o = p @ v
            else:
                o = torch.stack([(p[i][ok[i]][:, None] * v[ok[i]]).sum(dim=0) for i in range(p.shape[0])])
            size = p @ v.abs().nan_to_num(0, 0, 0)
            out[t, h], lse[h, t] = o, z
            # fp32: a score is a sum of d products (error at most (d + 4) half steps of the sum of their sizes, which the reference of the
            # exponentials has once more), O and l are sums of as many terms as there are keys; each p is rounded to the storage type,
            # and O in the end; p below fp16's normal range is off by half its smallest step
            sizes = torch.where(ok, q.abs() @ k.abs().nan_to_num(0, 0, 0).T * c.scale, 0.0).amax(dim=1)
            c32 = 2 * ((d + 4) * 2 * sizes + ok.sum(dim=1) + 8) * 2.0 ** -24
            tol[t, h] = u * o.abs().nan_to_num(0, 0, 0) + (u + c32[:, None]) * size * (1 + u)
            if c.dtype == "fp16":
                tol[t, h] += 2.0 ** -25 * (1 + (ok.double() @ v.abs().nan_to_num(0, 0, 0)))
            tol_lse[h, t] = c32 + 2.0 ** -22 * (z.abs().nan_to_num(0, 0, 0) + top.abs().nan_to_num(0, 0, 0))
    return out, lse, tol, tol_lse


def weights(c, lse):
    """(scores [pages, kv_heads, page] of one call that found zeros, how far off) for the lse that the call is given."""
    scores = torch.zeros(c.pages, c.kv_heads, c.page, dtype=torch.float64)
    tol = torch.zeros_like(scores)
    group = c.heads // c.kv_heads
    for b in range(len(c.lens)):
        if not c.news[b] or not c.lens[b]:
            continue
        t = slice(int(c.starts[b]), int(c.starts[b + 1]))
        for g in range(c.kv_heads):
            k, there = c.rows(c.k, b, g)
            ok = c.seen(b, there)
            w, off = torch.zeros(c.lens[b], dtype=torch.float64), torch.zeros(c.lens[b], dtype=torch.float64)
            for h in range(g * group, (g + 1) * group):
                q, z = c.q[t, h].double(), lse[h, t].double()
                use = ok & (z != -math.inf)[:, None]
                s = q @ k.T * c.scale
                p = torch.where(use, torch.exp(s - z[:, None]), 0.0)
                sizes = q.abs() @ k.abs().T * c.scale
                # the exponent is off as a score is, and by the rounding of lse log2(e) and of the difference; then a sum over the rows
                e = ((c.dim + 4) * sizes + 4 * z.abs().nan_to_num(0, 0, 0)[:, None] + 4 * s.abs() + 8 + use.sum(dim=0)[None, :] * group) * 2.0 ** -24
                w += p.sum(dim=0)
                off += torch.where(use, 2 * e * p, 0.0).sum(dim=0)
            for j in range(c.lens[b]):
                page = c.row(b, j)
                if page is not None:
                    scores[page, g, j % c.page] = w[j]
                    tol[page, g, j % c.page] = off[j] + 2.0 ** -126
    return scores, tol


def kept(scores, there, budget, first, last):
    """Places that stay of one sequence's KV head: scores [L], there [L]."""
    L = len(scores)
    if L <= budget:
        return list(range(L))
    value = [(-math.inf if math.isnan(x) or not t else x) for x, t in zip(scores.tolist(), there.tolist())]
    middle = sorted(range(first, L - last), key=lambda j: (-value[j], j))[:budget - first - last]
    return sorted(list(range(first)) + middle + list(range(L - last, L)))
