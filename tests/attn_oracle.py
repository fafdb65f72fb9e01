"""Attention and cache bookkeeping from their definitions, in 64 bits on the host, and the error a
kernel may make."""
from __future__ import annotations

import numpy as np
import torch

# Unit roundoffs of the activation types and of fp32.
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U32 = 2.0 ** -24


def attend(q, k, v, limits, scale, dtype):
    """Rows q [n, D] over keys [0, limits[r]) of k, v [m, D] (any values past the limits): (out, lse, bound on
    |out error|, bound on |lse error|) in float64.

    The bounds: a score's fp32 sum of D products is off by at most (D + 2) U32 times the sum of their
    magnitudes (delta below, with the exponential's own 2^-21); that moves every weight by a factor of at
    most exp(2 delta) against the others. Each weight is rounded once to the activation type (U; in fp16
    a weight below 2^-14 of the largest by at most 2^-25 of it), the output once; sums over m keys add m U32."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    n, D = q.shape
    limits = torch.as_tensor(limits).long()
    m = limits.clamp(min=0).double()
    seen = torch.arange(k.shape[0])[None, :] < limits[:, None]
    u = U[dtype]
    s = torch.where(seen, (q @ k.T) * scale, -np.inf)
    mag = torch.where(seen, (q.abs() @ k.abs().T) * scale, 0.0)
    none = ~seen.any(1)
    if none.all():
        z = torch.zeros(n, D, dtype=torch.float64)
        return z, torch.full((n,), -np.inf, dtype=torch.float64), z, z[:, 0]
    top = torch.where(none, 0.0, s.max(1).values)
    p = torch.where(seen, torch.exp(s - top[:, None]), 0.0)
    l = torch.where(none, 1.0, p.sum(1))
    p = p / l[:, None]

    def weigh(x):  # sum over the keys a row sees; others take no part, even where they are not finite
        y = p @ torch.where(torch.isfinite(x), x, 0.0)
        for j in torch.nonzero(~torch.isfinite(x).all(1)).flatten().tolist():
            y += torch.where(seen[:, j, None] & ~torch.isfinite(x[j]), p[:, j, None] * x[j], 0.0)
        return y

    out = weigh(v)
    lse = torch.where(none, -np.inf, top + torch.log(l))
    delta = (D + 2) * U32 * mag.max(1).values + 2.0 ** -21
    vabs = torch.where(torch.isfinite(v), v.abs(), 0.0)
    ob = u * out.abs() + (u + 2 * delta + (m + 64) * U32)[:, None] * (p @ vabs)
    if dtype == torch.float16:
        ob += 2.0 ** -24 + (m * 2.0 ** -25 / l)[:, None] * vabs.max()
    lb = delta + (m + 64) * U32 + 4 * U32 * (1 + torch.where(none, 0.0, lse.abs()))
    return out, lse, 1.01 * ob, 1.01 * lb


def check(got, lse, want, label=""):
    """got [n, D] (and lse [n] or None) against attend()'s answer."""
    out, ref_lse, ob, lb = want
    got = got.double().cpu()
    f = torch.isfinite(out)
    assert torch.equal(torch.isfinite(got), f), f"{label}: non-finite outputs"
    assert torch.equal(torch.isnan(got), torch.isnan(out)) and torch.equal(got[~f & ~torch.isnan(out)], out[~f & ~torch.isnan(out)]), label
    got, out, ob = got[f], out[f], ob[f]
    over = ((got - out).abs() - ob).max().item() if got.numel() else 0.0
    worst = ((got - out).abs() / ob.clamp(min=1e-30)).max().item() if got.numel() else 0.0
    assert over <= 0, f"{label}: off by {worst:.3g} of the bound"
    if lse is not None:
        lse = lse.double().cpu()
        assert torch.equal(torch.isneginf(lse), torch.isneginf(ref_lse)), label
        f = torch.isfinite(ref_lse)
        d = ((lse - ref_lse)[f].abs() - lb[f])
        assert d.numel() == 0 or d.max().item() <= 0, f"{label}: lse off by {((lse - ref_lse)[f].abs() / lb[f]).max():.3g} of the bound"
    return worst


class Cache:
    """The cache's table, lengths and counts by the rules of include/hq_attn.h, and its pools on the host."""

    def __init__(self, k, v, table, lens, refs):
        self.k, self.v = k.clone(), v.clone()  # [layers, pages, heads, tokens, dim]
        self.table, self.lens, self.refs = (np.array(x, dtype=np.int64) for x in (table, lens, refs))
        self.T = k.shape[3]

    def lowest_free(self):
        free = np.flatnonzero(self.refs == 0)
        return int(free[0]) if len(free) else None

    def reserve(self, rows, counts):
        save = self.table.copy(), self.lens.copy(), self.refs.copy()
        for r, c in zip(rows, counts):
            want = self.lens[r] + c
            have, need = -(-self.lens[r] // self.T), -(-want // self.T)
            if need > self.table.shape[1]:
                self.table, self.lens, self.refs = save
                return "full"
            for j in range(have, need):
                p = self.lowest_free()
                if p is None:
                    self.table, self.lens, self.refs = save
                    return "pages"
                self.table[r, j] = p
                self.refs[p] = 1
            self.lens[r] = want

    def append(self, layer, k, v, rows, cu):
        for i, r in enumerate(rows):
            n = cu[i + 1] - cu[i]
            for t in range(n):
                at = self.lens[r] - n + t
                p = self.table[r, at // self.T]
                self.k[layer, p, :, at % self.T] = k[cu[i] + t]
                self.v[layer, p, :, at % self.T] = v[cu[i] + t]

    def fork(self, parents, children):
        for p, c in zip(parents, children):
            full, part = divmod(int(self.lens[p]), self.T)
            self.table[c] = -1
            for j in range(full):
                self.table[c, j] = self.table[p, j]
                self.refs[self.table[p, j]] += 1
            if part:
                new = self.lowest_free()
                src = self.table[p, full]
                for pool in (self.k, self.v):
                    pool[:, new, :, :part] = pool[:, src, :, :part]
                self.table[c, full] = new
                self.refs[new] = 1
            self.lens[c] = self.lens[p]

    def free(self, rows):
        for r in rows:
            for j in range(-(-int(self.lens[r]) // self.T)):
                self.refs[self.table[r, j]] -= 1
                self.table[r, j] = -1
            self.lens[r] = 0

    def compact(self):
        live = np.flatnonzero(self.refs > 0)
        n = len(live)
        holes, movers = np.flatnonzero(self.refs[:n] == 0), live[live >= n]
        to = np.arange(len(self.refs))
        for s, d in zip(movers, holes):
            to[s] = d
            self.refs[d], self.refs[s] = self.refs[s], 0
            for pool in (self.k, self.v):
                pool[:, d] = pool[:, s]
        self.table = np.where(self.table >= 0, to[np.maximum(self.table, 0)], self.table)

    def tokens(self, pool, layer, row, head, n=None):
        """The first n tokens of a row, one head: [n, dim]."""
        n = int(self.lens[row]) if n is None else n
        pages = self.table[row, :-(-n // self.T)]
        return pool[layer, torch.from_numpy(pages), head].reshape(-1, pool.shape[-1])[:n]
