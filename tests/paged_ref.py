"""Plain 64-bit restatements of the rotary and paged-cache operators, and a
fixture that holds a cache in torch tensors registered with a session."""
import math

import numpy as np
import torch

from fercuda_b200 import capi

CODES = {torch.float32: capi.FER_DTYPE_F32, torch.float16: capi.FER_DTYPE_F16, torch.bfloat16: capi.FER_DTYPE_BF16,
         torch.int32: capi.FER_DTYPE_I32, torch.uint8: capi.FER_DTYPE_U8}


def half_step(ref, dtype):
    """The most that rounding a value to dtype can change it (float64 tensors)."""
    f = torch.finfo(dtype)
    return (ref.abs() * (f.eps / 2)).clamp(min=f.smallest_normal * f.eps / 2)


class Buffers:
    """Registers tensors with a session on torch's current stream; frees the ids at the end."""

    def __init__(self, session):
        self.s, self.ids, self.keep = session, [], []

    def __enter__(self):
        self.before = self.s.stream()
        self.s.set_stream(torch.cuda.current_stream().cuda_stream)
        return self

    def __exit__(self, *exc):
        torch.cuda.synchronize()
        for i in self.ids:
            self.s.free(i)
        self.s.set_stream(self.before)

    def __call__(self, t):
        if t is None:
            return 0
        assert t.is_contiguous()
        self.keep.append(t)
        self.ids.append(self.s.import_ptr(CODES[t.dtype], list(t.shape), t.data_ptr()))
        return self.ids[-1]

    def workspace(self, size):
        """Any contents: all ones, so that floats in it are NaN."""
        return self(torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda"))


class Cache:
    """Pages full of NaN but for the held slots, a table whose entries behind
    them are no page ids, and weights and positions that hold a mark where
    nothing may be written."""

    def __init__(self, lengths, kv_heads, head_dim, page, dtype, max_pages=None, seed=0, spare=2):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.H, self.D, self.P, self.dtype = list(lengths), kv_heads, head_dim, page, dtype
        B = len(self.lens)
        need = [-(-n // page) for n in self.lens]
        self.max_pages = max_pages or max(1, max(need))
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g).tolist()
        table = torch.full((B, self.max_pages), -7, dtype=torch.int32)
        table[:, 1::2] = 10 ** 9
        k = torch.full((pages, kv_heads, page, head_dim), math.nan, dtype=dtype)
        v = k.clone()
        for b, n in enumerate(self.lens):
            for i in range(need[b]):
                p = table[b, i] = order.pop()
                m = min(page, n - i * page)
                k[p, :, :m] = torch.randn(kv_heads, m, head_dim, generator=g).to(dtype)
                v[p, :, :m] = torch.randn(kv_heads, m, head_dim, generator=g).to(dtype)
        self.k, self.v, self.table = k.cuda(), v.cuda(), table.cuda()
        self.lengths = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.slots = self.max_pages * page

    def ids(self, bufs):
        return capi.paged_cache(bufs(self.k), bufs(self.v), bufs(self.table), bufs(self.lengths))

    def rows(self, pool, b, h, n=None):
        """Rows of the held slots of (b, h), float64 on the CPU."""
        n = self.lens[b] if n is None else n
        s = torch.arange(n)
        page = self.table.cpu()[b, s // self.P].long()
        return pool.cpu()[page, h, s % self.P].double()


def attention(cache, q, heads, scale=None, skip=None):
    """out [B, heads, D], lse, the probabilities' sums per (b, kv head), and
    the bound of the absolute error before rounding, all float64."""
    D, group = cache.D, heads // cache.H
    scale = D ** -0.5 if scale is None else scale
    q = q.cpu().double().view(-1, heads, D)
    B = q.shape[0]
    out, lse = torch.zeros(B, heads, D, dtype=torch.float64), torch.full((B, heads), -math.inf, dtype=torch.float64)
    err, sums = torch.zeros_like(out), {}
    for b in range(B):
        for h in range(cache.H):
            k, v = cache.rows(cache.k, b, h), cache.rows(cache.v, b, h)
            held = torch.ones(k.shape[0], dtype=torch.bool)
            if skip:
                held[[s for (bb, s) in skip if bb == b]] = False
            qq = q[b, h * group:(h + 1) * group]
            z = (qq @ k.T * scale)[:, held]
            if z.shape[1] == 0 or bool((z == -math.inf).all()):
                sums[b, h] = torch.zeros(k.shape[0], dtype=torch.float64), 0.0
                continue
            top = z.amax(1, keepdim=True)
            e = torch.exp(z - top)
            p = e / e.sum(1, keepdim=True)
            sl = slice(h * group, (h + 1) * group)
            out[b, sl] = p @ v[held]
            lse[b, sl] = (top + e.sum(1, keepdim=True).log())[:, 0]
            w = torch.zeros(k.shape[0], dtype=torch.float64)
            w[held] = p.sum(0)
            # a score in f32: products exact, D additions and the scaling, each at most 2^-23 of the
            # absolute products' sum; an exponent of its size again; p and l by twice that; p itself
            # kept to 16 bits or more, and the sum over v in f32
            ds = float((qq.abs() @ k[held].abs().T * scale).max()) * (D + 4) * 2.0 ** -23
            rel = 2 * ds + 2.0 ** -16 + z.shape[1] ** 0.5 * 2.0 ** -23
            err[b, sl] = rel * (p @ v[held].abs())
            sums[b, h] = w, 2 * ds + 2.0 ** -20
    return out, lse, sums, err


def evict(weights, positions, n, budget, recent, seen):
    """(kept slots that stay, list of (from, to)) of one (sequence, key head), numpy arrays in."""
    if n <= budget:
        return list(range(n)), []
    def rank(i):
        if positions[i] >= seen - recent:
            return (0, 0.0, i)
        w = float(weights[i])
        return (2, 0.0, i) if math.isnan(w) else (1, -w, i)
    kept = sorted(sorted(range(n), key=rank)[:budget])
    free = sorted(set(range(budget)) - set(kept))
    return [i for i in kept if i < budget], list(zip([i for i in kept if i >= budget], free))


def rotary(x, positions, heads, head_dim, sections, rotary_dim, base, interleaved, axis_freqs, inverse):
    """float64 [rows, heads, head_dim] from x [rows, heads * head_dim], and the pairs' (cos, sin) angles' bound."""
    x = x.double().view(x.shape[0], heads, head_dim)
    y = x.clone()
    half, i = rotary_dim // 2, 0
    far = torch.zeros(x.shape[0], dtype=torch.float64)
    for a, n in enumerate(sections):
        for j in range(n):
            f = base ** -(j / n if axis_freqs else i / half)
            t = positions[:, a].double() * (-f if inverse else f)
            far = torch.maximum(far, t.abs())
            c, s = t.cos()[:, None], t.sin()[:, None]
            u, w = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            y[:, :, u], y[:, :, w] = x[:, :, u] * c - x[:, :, w] * s, x[:, :, u] * s + x[:, :, w] * c
            i += 1
    return y, far


def as_np(t):
    return t.detach().cpu().numpy() if t.dtype != torch.bfloat16 else t.detach().float().cpu().numpy()


def same_bits(a, b):
    return np.array_equal(a.contiguous().view(torch.uint8).cpu().numpy(), b.contiguous().view(torch.uint8).cpu().numpy())
