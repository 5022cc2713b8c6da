"""64-bit restatements of windowed and shared-prefix attention over a paged cache,
with a bound of the absolute error before the result is rounded.

A score in f32: products exact, D additions and the scaling, each at most 2^-23 of
the absolute products' sum (ds). A probability: an exponent off by 2 ds, the
exponential by 2^-18 (a polynomial of relative error 2.9e-6 with f32 arithmetic,
or the hardware's, which is better), rounded to the type once, half a step of it
(where a unit has few rows it is kept to twice the bits, which is less). Sums of
n terms in f32: at most sqrt(n) 2^-23 beside the rest here."""
import math

import torch


def rows_of(lens, offsets, group):
    """(row, sequence, slot) of every row that belongs to a sequence."""
    if offsets is None:
        return [(b, b, n - 1) for b, n in enumerate(lens)]
    return [(r, b, lens[b] - (offsets[b + 1] - offsets[b]) + r - offsets[b])
            for b in range(len(offsets) - 1) for r in range(offsets[b], offsets[b + 1])]


def softmax_rows(q, k, v, seen, scale, dtype):
    """q [G, D], k and v [n, D], seen [n]: out [G, D], lse [G], err [G, D], ds."""
    D = q.shape[1]
    k, v = k[seen], v[seen]
    z = q @ k.T * scale
    if z.shape[1] == 0 or bool((z == -math.inf).all()):
        return torch.zeros_like(q), torch.full((q.shape[0],), -math.inf, dtype=torch.float64), torch.zeros_like(q), 0.0
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    p = e / e.sum(1, keepdim=True)
    ds = float((q.abs() @ k.abs().T * scale).max()) * (D + 4) * 2.0 ** -23
    rel = 2 * ds + 2.0 ** -18 + torch.finfo(dtype).eps / 2 + z.shape[1] ** 0.5 * 2.0 ** -23
    return p @ v, (top + e.sum(1, keepdim=True).log())[:, 0], rel * (p @ v.abs()), 2 * ds + 2.0 ** -17


def window(c, q, heads, offsets, win, sinks, scale=None, skip=()):
    """out and err [rows, heads, D], lse [rows, heads], the lse's bound; rows of no sequence are NaN. skip: (sequence, slot)."""
    group, scale = heads // c.H, c.D ** -0.5 if scale is None else scale
    q = q.cpu().double().view(-1, heads, c.D)
    out = torch.full_like(q, math.nan)
    err, lse, most = torch.zeros_like(q), torch.full(q.shape[:2], math.nan, dtype=torch.float64), 0.0
    for h in range(c.H):
        kv = [(c.rows(c.k, b, h), c.rows(c.v, b, h)) for b in range(len(c.lens))]
        for r, b, at in rows_of(c.lens, offsets, group):
            k, v = kv[b]
            s = torch.arange(k.shape[0])
            seen = s <= at
            if win:
                seen &= (s > at - win) | (s < sinks)
            for (bb, x) in skip:
                if bb == b:
                    seen[x] = False
            sl = slice(h * group, (h + 1) * group)
            out[r, sl], lse[r, sl], err[r, sl], ds = softmax_rows(q[r, sl], k, v, seen, scale, c.dtype)
            most = max(most, ds)
    return out, lse, err, most


def prefix(c, pages, length, q, heads, scale=None):
    """The same behind `length` slots of the pages of c's pools."""
    group, scale = heads // c.H, c.D ** -0.5 if scale is None else scale
    q = q.cpu().double().view(-1, heads, c.D)
    out, err = torch.zeros_like(q), torch.zeros_like(q)
    lse, most = torch.zeros(q.shape[:2], dtype=torch.float64), 0.0
    s = torch.arange(length)
    at = torch.as_tensor(pages)[s // c.P].long() if length else s
    for h in range(c.H):
        pk, pv = c.k.cpu()[at, h, s % c.P].double(), c.v.cpu()[at, h, s % c.P].double()
        for b in range(q.shape[0]):
            k, v = torch.cat([pk, c.rows(c.k, b, h)]), torch.cat([pv, c.rows(c.v, b, h)])
            sl = slice(h * group, (h + 1) * group)
            out[b, sl], lse[b, sl], err[b, sl], ds = softmax_rows(q[b, sl], k, v, torch.ones(len(k), dtype=torch.bool), scale, c.dtype)
            most = max(most, ds)
    return out, lse, err, most
