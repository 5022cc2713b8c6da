"""The paged-cache operators (fer_submit_paged_store, fer_submit_paged_attention,
fer_submit_paged_evict and their launchers) against 64-bit restatements.

Copies and selections are exact. Attention is held to half a step of its type
plus the arithmetic bound that tests/paged_ref.py derives; lse and weights to
that bound in f32. Pages are NaN outside the held slots, and table entries
behind them are no page ids, so anything that is read there shows."""
import copy
import ctypes as C
import math
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from fercuda_b200 import capi
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
ERR_BAD = 4


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def attend(session, c, q, heads, weights=None, q_col=0, out=None, out_col=0, scale=0.0, errors=0):
    rows = q.shape[0]
    out = torch.full((rows, heads * c.D), 7.0, dtype=c.dtype, device="cuda") if out is None else out
    lse = torch.full((rows, heads), 7.0, device="cuda")
    with ref.Buffers(session) as B:
        size = capi.paged_attention_workspace_bytes(rows, heads, c.H, c.D, c.slots, weights is not None)
        bq = B(q)
        session.paged_attention(c.ids(B), bq, bq if out is q else B(out), heads, workspace=B.workspace(size),
                                q_col=q_col, out_col=out_col, scale=scale, lse=B(lse), weights=B(weights))
    assert session.device_errors() == errors
    return out, lse


def check(c, q, heads, out, lse, scale=None, skip=None):
    want, wlse, sums, err = ref.attention(c, q, heads, scale, skip)
    got = out.cpu().double().view_as(want)
    assert bool(((got - want).abs() <= ref.half_step(want, c.dtype) + err).all()), float((got - want).abs().max())
    some = wlse > -math.inf
    assert torch.equal(lse.cpu() > -math.inf, some)
    ds = max((s[1] for s in sums.values()), default=0.0)
    assert bool(((lse.cpu().double() - wlse)[some].abs() <= ds + wlse[some].abs() * 2.0 ** -21 + 2.0 ** -20).all())
    return sums


def queries(c, heads, rows=None, seed=1, factor=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows or len(c.lens), heads * c.D, generator=g) * factor).to(c.dtype).cuda()


# ------------------------------------------------------------------ attention

@pytest.mark.parametrize("dtype,D,H,group,page,lens", [
    (BF16, 64, 1, 1, 16, [1]),
    (BF16, 64, 2, 1, 8, [0, 1, 2, 7, 8, 9, 63, 64, 65]),
    (F16, 64, 3, 2, 32, [255, 256, 257, 31, 0]),
    (F16, 128, 2, 3, 16, [511, 512, 513]),
    (BF16, 128, 1, 5, 64, [127, 128, 129, 0, 1]),
    (F16, 128, 2, 4, 128, [1000, 17]),
    (BF16, 128, 1, 8, 16, [300, 15, 16]),
    (F16, 64, 1, 16, 256, [257, 1025]),
    (BF16, 64, 1, 17, 16, [333, 48]),
    (BF16, 128, 2, 24, 8, [100, 99]),
    (BF16, 64, 1, 71, 32, [77]),
    (F16, 256, 2, 1, 16, [1, 40, 129]),
    (BF16, 256, 1, 6, 64, [511, 0, 65]),
    (BF16, 256, 1, 12, 8, [70]),
    (F16, 64, 16, 1, 16, [600] * 9)])
def test_attention(session, dtype, D, H, group, page, lens):
    c = ref.Cache(lens, H, D, page, dtype, seed=D + H + group)
    q = queries(c, H * group)
    check(c, q, H * group, *attend(session, c, q, H * group))


@pytest.mark.parametrize("dtype,D,H,group,page,lens,width", [
    (BF16, 64, 2, 1, 16, [0, 1, 16, 17, 300], None),
    (F16, 128, 1, 4, 32, [513, 5], 64),
    (BF16, 128, 2, 3, 8, [65, 640], 200),
    (F16, 64, 1, 19, 64, [130], 3),
    (BF16, 256, 1, 2, 16, [33, 4], None),
    (BF16, 64, 2, 2, 128, [5000, 4097], 300)])
def test_attention_weights(session, dtype, D, H, group, page, lens, width):
    c = ref.Cache(lens, H, D, page, dtype, max_pages=width, seed=3)
    q = queries(c, H * group)
    before = torch.rand(len(lens), H, c.slots, generator=torch.Generator().manual_seed(5))
    for b, n in enumerate(lens):
        before[b, :, n:] = math.nan
    w = before.cuda()
    sums = check(c, q, H * group, *attend(session, c, q, H * group, weights=w))
    w2 = before.cuda()
    attend(session, c, q, H * group, weights=w2)
    assert ref.same_bits(w, w2)
    for b, n in enumerate(lens):
        assert bool(torch.isnan(w[b, :, n:]).all())
        for h in range(H):
            want, rel = sums[b, h]
            now = w[b, h, :n].cpu().double()
            total = want + before[b, h, :n].double()
            assert bool(((now - total).abs() <= want * rel + total * 2.0 ** -23).all())


def test_attention_scale(session):
    c = ref.Cache([90, 7], 2, 64, 16, BF16)
    q = queries(c, 4)
    check(c, q, 4, *attend(session, c, q, 4, scale=0.37), scale=float(np.float32(0.37)))


@pytest.mark.parametrize("q_col,out_col", [(0, 64 * 6), (3, 5), (8, 16)])
def test_attention_columns_of_a_fused_activation(session, q_col, out_col):
    c = ref.Cache([70, 33, 1], 2, 64, 16, F16)
    heads, width = 6, 64 * 6
    wide = queries(c, 20, seed=9)
    if q_col == 0:
        out = wide                                         # one buffer, columns apart
    else:
        out = torch.full((3, width + 24), 7.0, dtype=F16, device="cuda")
    q = wide[:, q_col:q_col + width].clone()
    rest = out.clone()
    attend(session, c, wide, heads, q_col=q_col, out=out, out_col=out_col)
    part = out[:, out_col:out_col + width].contiguous()
    alone, lse = attend(session, c, q.contiguous(), heads)
    check(c, q, heads, alone, lse)
    assert ref.same_bits(part, alone)
    out[:, out_col:out_col + width] = rest[:, out_col:out_col + width]
    assert ref.same_bits(out, rest)


@pytest.mark.parametrize("page,group", [(16, 1), (64, 4)])
def test_a_sequence_does_not_depend_on_its_batch(session, page, group):
    lens = [700, 3, 0, 256, 1300, 511]
    c = ref.Cache(lens, 2, 128, page, BF16)
    q = queries(c, 2 * group)
    w = torch.zeros(len(lens), 2, c.slots, device="cuda")
    out, lse = attend(session, c, q, 2 * group, weights=w)
    again = attend(session, c, q, 2 * group, weights=torch.zeros_like(w))
    assert ref.same_bits(out, again[0]) and ref.same_bits(lse, again[1])
    for b in range(len(lens)):
        one = ref.Cache([lens[b]], 2, 128, page, BF16)
        one.k, one.v, one.table, one.lengths = c.k, c.v, c.table[b:b + 1].clone(), c.lengths[b:b + 1].clone()
        one.max_pages, one.slots = c.max_pages, c.slots
        w1 = torch.zeros(1, 2, c.slots, device="cuda")
        o1, l1 = attend(session, one, q[b:b + 1].clone(), 2 * group, weights=w1)
        assert ref.same_bits(o1, out[b:b + 1]) and ref.same_bits(l1, lse[b:b + 1]) and ref.same_bits(w1, w[b:b + 1])


@pytest.mark.parametrize("dtype,D,H,group,page,B,most", [
    (BF16, 64, 8, 1, 16, 300, 700),      # more units than CTAs, segments of three sequences
    (F16, 128, 4, 4, 32, 130, 1100),
    (BF16, 256, 2, 12, 64, 129, 600),
    (BF16, 64, 1, 20, 8, 1000, 40),
    (F16, 128, 2, 16, 128, 150, 600)])
def test_attention_of_large_ragged_batches(session, dtype, D, H, group, page, B, most):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, most + 1, (B,), generator=g)
    lens[torch.rand(B, generator=g) < 0.2] = 0             # runs of empty sequences, the first and last among them
    lens[:2] = lens[-3:] = 0
    lens = lens.tolist()
    lens[B // 2] = most
    c = ref.Cache(lens, H, D, page, dtype, seed=B)
    q = queries(c, H * group)
    w = torch.zeros(B, H, c.slots, device="cuda")
    out, lse = attend(session, c, q, H * group, weights=w)
    host = copy.copy(c)
    host.k, host.v, host.table = c.k.cpu(), c.v.cpu(), c.table.cpu()
    sums = check(host, q, H * group, out, lse)
    now = w.cpu().double()
    for (b, h), (want, rel) in sums.items():
        assert bool(((now[b, h, :lens[b]] - want).abs() <= want * (rel + 2.0 ** -23) + 2.0 ** -140).all())
        assert not now[b, h, lens[b]:].any()
    b = B // 2
    one = ref.Cache([most], H, D, page, dtype)
    one.k, one.v, one.table, one.lengths = c.k, c.v, c.table[b:b + 1].clone(), c.lengths[b:b + 1].clone()
    o1, l1 = attend(session, one, q[b:b + 1].clone(), H * group)
    assert ref.same_bits(o1, out[b:b + 1]) and ref.same_bits(l1, lse[b:b + 1])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_of_short_sequences_in_a_wide_table(session, D):
    lens = torch.randint(0, 300, (100,), generator=torch.Generator().manual_seed(3)).tolist()
    lens[7], lens[50] = 12001, 1025
    c = ref.Cache(lens, 4, D, 64, BF16, max_pages=256)
    q = queries(c, 8)
    w = torch.zeros(100, 4, c.slots, device="cuda")
    out, lse = attend(session, c, q, 8, weights=w)
    host = copy.copy(c)
    host.k, host.v, host.table = c.k.cpu(), c.v.cpu(), c.table.cpu()
    sums = check(host, q, 8, out, lse)
    now = w.cpu().double()
    for (b, h), (want, rel) in sums.items():
        assert bool(((now[b, h, :lens[b]] - want).abs() <= want * (rel + 2.0 ** -23) + 2.0 ** -140).all())
        assert not now[b, h, lens[b]:].any()
    for b in (7, 50, 51):                                  # alone in the same table: the same bits
        one = copy.copy(c)
        one.lens, one.table, one.lengths = lens[b:b + 1], c.table[b:b + 1].clone(), c.lengths[b:b + 1].clone()
        w1 = torch.zeros(1, 4, c.slots, device="cuda")
        o1, l1 = attend(session, one, q[b:b + 1].clone(), 8, weights=w1)
        assert ref.same_bits(o1, out[b:b + 1]) and ref.same_bits(l1, lse[b:b + 1]) and ref.same_bits(w1, w[b:b + 1])


def test_attention_of_a_large_batch_that_holds_nothing(session):
    c = ref.Cache([0] * 700, 2, 64, 16, BF16, max_pages=40)
    out, lse = attend(session, c, queries(c, 4), 4)
    assert not out.any() and bool((lse == -math.inf).all())


def test_bad_pages_in_a_large_batch(session):
    """As above, where a CTA has several units."""
    lens = [300] * 200
    c = ref.Cache(lens, 4, 64, 16, BF16)
    q = queries(c, 4)
    good, gl = attend(session, c, q, 4)
    c.table[70, 17] = -1                                   # a page of the second chunk
    c.table[199, :19] = 10 ** 6
    out, lse = attend(session, c, q, 4, errors=ERR_BAD)
    others = [b for b in range(200) if b not in (70, 199)]
    assert ref.same_bits(out[others], good[others]) and ref.same_bits(lse[others], gl[others])
    assert not out[199].any() and bool((lse[199] == -math.inf).all())
    one = copy.copy(c)
    one.lens, one.table = [300], c.table[70:71].clone()
    one.table[0, 17] = c.table[0, 0]                       # any page: the oracle leaves those slots out
    check(one, q[70:71], 4, out[70:71], lse[70:71], skip={(0, s) for s in range(272, 288)})


def test_fewer_rows_than_the_cache_has_sequences(session):
    c = ref.Cache([70, 33, 300], 2, 64, 16, F16)
    q = queries(c, 2)
    out, _ = attend(session, c, q, 2)
    two, _ = attend(session, c, q[:2].clone(), 2)
    assert ref.same_bits(two, out[:2])


def test_infinities_and_nan(session):
    """-inf scores count as nothing, also all of them; inf and NaN reach their own heads and no others."""
    c = ref.Cache([300, 300, 300, 20], 2, 64, 16, BF16)
    at = lambda b, s: (int(c.table[b, s // 16]), s % 16)   # noqa: E731
    p, r = at(0, 270)
    c.k[p, 0, r] = torch.tensor([-math.inf] + [0.0] * 63)  # q[0] > 0 there: one score -inf
    p, r = at(1, 3)
    c.v[p, 1, r] = math.inf                                # a value inf
    p, r = at(2, 299)
    c.k[p, 1, r, 5] = math.nan                             # a score NaN
    for s in range(20):
        p, r = at(3, s)
        c.k[p, 0, r] = torch.tensor([-math.inf] + [0.0] * 63)
    q = queries(c, 2)
    q[:, 0] = 1.0
    w = torch.zeros(4, 2, c.slots, device="cuda")
    out, lse = attend(session, c, q, 2, weights=w)
    o = out.view(4, 2, 64)
    assert bool(torch.isfinite(o[0]).all()) and float(w[0, 0, 270]) == 0.0
    assert bool((o[1, 1] == math.inf).all()) and bool(torch.isfinite(o[1, 0]).all())
    assert bool(torch.isnan(o[2, 1]).all()) and bool(torch.isfinite(o[2, 0]).all())
    assert bool((o[3, 0] == 0).all()) and float(lse[3, 0]) == -math.inf and bool((w[3, 0] == 0).all())
    assert bool(torch.isfinite(o[3, 1]).all())
    want, wlse, _, err = ref.attention(c, q, 2)
    for b, h in ((0, 0), (0, 1), (1, 0), (2, 0), (3, 1)):
        assert bool(((o[b, h].cpu().double() - want[b, h]).abs()
                     <= ref.half_step(want[b, h], BF16) + err[b, h]).all()), (b, h)


def test_scores_of_lowest_and_largest_values(session):
    """Scores of +-1e4 and a spread that underflows: the maximum alone is left."""
    c = ref.Cache([400], 1, 64, 32, BF16)
    c.k.copy_(torch.nan_to_num(c.k) * 0)
    p = c.table[0, 350 // 32]
    c.k[c.table[0, 0], 0, 3, 0] = -100.0
    c.k[p, 0, 350 % 32, 0] = 100.0
    q = torch.zeros(1, 64, dtype=BF16, device="cuda")
    q[0, 0] = 800.0
    out, lse = attend(session, c, q, 1)
    assert ref.same_bits(out[0], c.v[p, 0, 350 % 32])
    assert abs(float(lse[0, 0]) - 1e4) <= 1e4 * 2.0 ** -22


def test_pages_may_be_shared_for_reading(session):
    c = ref.Cache([100, 100], 2, 64, 16, F16)
    c.table[1] = c.table[0]
    c.table[1, 2] = c.table[0, 0]                          # and a page may be there twice
    q = queries(c, 2)
    w = torch.zeros(2, 2, c.slots, device="cuda")
    sums = check(c, q, 2, *attend(session, c, q, 2, weights=w))
    for (b, h), (want, rel) in sums.items():
        assert bool(((w[b, h, :100].cpu().double() - want).abs() <= want * (rel + 2.0 ** -23)).all())


@pytest.mark.parametrize("bad", [-1, -2 ** 31, 10 ** 6])
def test_bad_pages_and_lengths_are_reported(session, bad):
    c = ref.Cache([100, 40, 90], 1, 64, 16, BF16)
    c.table[0, 3] = bad
    skip = {(0, s) for s in range(48, 64)}
    q = queries(c, 2)
    w = torch.zeros(3, 1, c.slots, device="cuda")
    out, lse = attend(session, c, q, 2, weights=w, errors=ERR_BAD)
    keep = c.table.clone()
    c.table[0, 3] = keep[1, 0]                             # any page: the oracle leaves those slots out
    sums = check(c, q, 2, out, lse, skip=skip)
    assert bool((w[0, 0, 48:64] == 0).all())
    assert bool(((w[0, 0, :100].cpu().double() - sums[0, 0][0]).abs()
                 <= sums[0, 0][0] * (sums[0, 0][1] + 2.0 ** -23)).all())
    c.table[0, 3] = bad
    # a length that the table cannot hold, or a negative one
    c.lengths.copy_(i32([c.slots + 5, -3, 90]))
    out, lse = attend(session, c, q, 2, errors=ERR_BAD)
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())
    # nothing but bad pages counts as nothing held
    c.lengths.copy_(i32([100, 40, 90]))
    c.table[2] = bad
    out, lse = attend(session, c, q, 2, errors=ERR_BAD)
    assert bool((out[2] == 0).all()) and bool((lse[2] == -math.inf).all())


@pytest.mark.parametrize("group,D", [(1, 64), (8, 128)])
def test_long_cache(session, group, D):
    n = 70001
    c = ref.Cache([n, 40], 1, D, 64, BF16)
    q = queries(c, group)
    w = torch.zeros(2, 1, c.slots, device="cuda")
    sums = check(c, q, group, *attend(session, c, q, group, weights=w))
    for b, m in ((0, n), (1, 40)):
        want, rel = sums[b, 0]
        assert bool(((w[b, 0, :m].cpu().double() - want).abs() <= want * (rel + 2.0 ** -23) + 2.0 ** -140).all())


def test_page_ids_behind_two_to_the_31_elements(session):
    """The pools have more than 2^32 elements and the pages in use lie at their end."""
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB")
    c = ref.Cache([600], 8, 256, 256, BF16)
    pages = (1 << 32) // (8 * 256 * 256) + 3
    small = (c.k, c.v)
    c.k, c.v = (torch.empty(pages, 8, 256, 256, dtype=BF16, device="cuda") for _ in range(2))
    used = c.table[0, :3].long()
    for new, old in ((c.k, small[0]), (c.v, small[1])):
        new[-3:] = old[used]
    low = ref.Cache([600], 8, 256, 256, BF16)
    c.table[0, :3] = i32([pages - 3, pages - 2, pages - 1])
    q = queries(c, 8)
    out, lse = attend(session, c, q, 8)
    want, wl = attend(session, low, q, 8)
    assert ref.same_bits(out, want) and ref.same_bits(lse, wl)
    check(low, q, 8, want, wl)
    # eviction and store at such pages
    w = torch.rand(1, 8, c.slots, device="cuda")
    pos = torch.arange(c.slots, dtype=torch.int32, device="cuda").repeat(1, 8, 1)
    for x in (c, low):
        run_evict(session, x, 200, 20, w.clone(), pos.clone(), i32([600]))
        x.lengths.copy_(i32([600]))
    assert ref.same_bits(c.k[-3:], low.k[low.table[0, :3].long()])
    rows = torch.randn(1, 2 * 8 * 256, device="cuda").to(BF16)
    with ref.Buffers(session) as B:
        r = B(rows)
        session.paged_store(c.ids(B), r, r, v_col=8 * 256)
    assert torch.equal(c.v[-1, :, 600 % 256].reshape(-1), rows[0, 8 * 256:])


# ------------------------------------------------------------------ store

def expect_store(c, rows, k_col, v_col, offsets, n_seq, weights, positions, seen):
    """Host copies of everything after a store."""
    k, v, lengths = c.k.cpu().clone(), c.v.cpu().clone(), c.lengths.cpu().clone()
    w, p, s = weights.cpu().clone(), positions.cpu().clone(), seen.cpu().clone()
    width = c.H * c.D
    for b in range(n_seq):
        lo, hi = (offsets[b], offsets[b + 1]) if offsets else (b, b + 1)
        for i, r in enumerate(range(lo, hi)):
            slot = c.lens[b] + i
            if slot >= c.slots:
                continue
            w[b, :, slot], p[b, :, slot] = 0.0, int(seen[b]) + i
            page = int(c.table[b, slot // c.P])
            if 0 <= page < c.k.shape[0]:
                k[page, :, slot % c.P] = rows[r, k_col:k_col + width].view(c.H, c.D).cpu()
                v[page, :, slot % c.P] = rows[r, v_col:v_col + width].view(c.H, c.D).cpu()
        lengths[b] = min(c.lens[b] + hi - lo, c.slots)
        s[b] += hi - lo
    return k, v, lengths, w, p, s


def grow_table(c):
    """Gives every entry of the table a page of its own; new pages are NaN."""
    B = c.table.shape[0]
    more = torch.full((B * c.max_pages, c.H, c.P, c.D), math.nan, dtype=c.dtype, device="cuda")
    n = c.k.shape[0]
    c.k, c.v = torch.cat([c.k, more]), torch.cat([c.v, more])
    fresh = torch.arange(B * c.max_pages, dtype=torch.int32, device="cuda").view(B, -1) + n
    used = torch.arange(c.max_pages, device="cuda") * c.P < c.lengths[:, None]
    c.table = torch.where(used, c.table, fresh).contiguous()


@pytest.mark.parametrize("dtype,D,H,page,lens,offsets,tail,cols", [
    (BF16, 64, 2, 16, [0, 15, 16, 17], None, 0, (0, 128)),
    (F16, 128, 3, 8, [5] * 40, None, 0, (0, 3 * 128)),
    (F16, 64, 1, 8, [3, 0, 7], [0, 1, 1, 10], 4, (64, 0)),
    (BF16, 128, 2, 64, [60, 0, 100, 1], [2, 2, 300, 301, 450], 7, (0, 256)),
    (BF16, 256, 1, 16, [1, 2], [0, 33, 66], 0, (3, 261)),            # odd columns: no 16-byte pieces
    (F16, 64, 5, 256, [0], [0, 1000], 0, (8, 328)),
    (BF16, 64, 2, 16, [4, 4, 4], [0, 5], 2, (0, 128))])              # fewer sequences than the cache has
@pytest.mark.parametrize("in_place", [False, True])
def test_store(session, dtype, D, H, page, lens, offsets, tail, cols, in_place):
    new = [b - a for a, b in zip(offsets, offsets[1:])] if offsets else [1] * len(lens)
    width = max(-(-(n + m) // page) for n, m in zip(lens, new + [0] * len(lens))) + 1
    c = ref.Cache(lens, H, D, page, dtype, max_pages=width)
    grow_table(c)
    rows_n = offsets[-1] + tail if offsets else len(lens)
    rows = torch.randn(rows_n, 2 * H * D + 16, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    w = torch.full((len(lens), H, c.slots), 5.0, device="cuda")
    p = torch.full((len(lens), H, c.slots), -5, dtype=torch.int32, device="cuda")
    seen = c.lengths * 3 + 1
    want = expect_store(c, rows, *cols, offsets, len(new), w, p, seen)
    old_len, old_seen = c.lengths.clone(), seen.clone()
    new_len, new_seen = (c.lengths, seen) if in_place else (c.lengths.clone(), seen.clone())
    with ref.Buffers(session) as B:
        r, ids, bseen = B(rows), c.ids(B), B(seen)
        session.paged_store(ids, r, r, k_col=cols[0], v_col=cols[1], offsets=B(i32(offsets)) if offsets else 0,
                            new_lengths=0 if in_place else B(new_len), weights=B(w), positions=B(p), seen=bseen,
                            new_seen=0 if in_place else B(new_seen))
    assert session.device_errors() == 0
    for got, exp in zip((c.k, c.v, new_len, w, p, new_seen), want):
        assert ref.same_bits(got, exp)
    if not in_place:
        assert torch.equal(c.lengths, old_len) and torch.equal(seen, old_seen)


@pytest.mark.parametrize("n_seq,ragged,H,col", [(400, True, 2, 0), (5000, False, 2, 0), (400, True, 1, 0),
                                                (400, True, 1, 3), (3000, False, 3, 8)])
@pytest.mark.parametrize("in_place", [False, True])
def test_store_of_many_rows(session, n_seq, ragged, H, col, in_place):
    """More rows than a CTA takes, and runs of sequences that get none."""
    g = torch.Generator().manual_seed(n_seq)
    new = torch.randint(0, 30, (n_seq,), generator=g) * (torch.rand(n_seq, generator=g) < 0.8) if ragged else None
    offsets = [3] + (3 + new.cumsum(0)).tolist() if ragged else None
    lens = torch.randint(0, 34, (n_seq,), generator=g).tolist()
    c = ref.Cache(lens, H, 64, 16, BF16, max_pages=4)
    grow_table(c)
    n = offsets[-1] + 5 if ragged else n_seq
    cols = (col, col + 64 * H)
    rows = torch.randn(n, 128 * H + 8, generator=g).to(BF16).cuda()
    w = torch.full((n_seq, H, c.slots), 5.0, device="cuda")
    p = torch.full((n_seq, H, c.slots), -5, dtype=torch.int32, device="cuda")
    seen = c.lengths + 9
    want = expect_store(c, rows, *cols, offsets, n_seq, w, p, seen)
    new_len, new_seen = (c.lengths, seen) if in_place else (c.lengths.clone(), seen.clone())
    with ref.Buffers(session) as B:
        r = B(rows)
        ids, bseen = c.ids(B), B(seen)
        session.paged_store(ids, r, r, k_col=cols[0], v_col=cols[1], offsets=B(i32(offsets)) if ragged else 0,
                            new_lengths=0 if in_place else B(new_len), weights=B(w), positions=B(p), seen=bseen,
                            new_seen=0 if in_place else B(new_seen))
    assert session.device_errors() == 0
    for got, exp in zip((c.k, c.v, new_len, w, p, new_seen), want):
        assert ref.same_bits(got, exp)


def test_store_of_keys_and_values_alone(session):
    """No weights, no positions, keys and values in buffers of their own."""
    c = ref.Cache([10, 31], 2, 64, 16, BF16, max_pages=3)
    grow_table(c)
    k, v = (torch.randn(2, 128, device="cuda").to(BF16) for _ in range(2))
    dummy = torch.zeros(2, 2, c.slots, device="cuda")
    both = torch.cat([k, v], 1)
    want = expect_store(c, both, 0, 128, None, 2, dummy, dummy.int(), c.lengths)
    with ref.Buffers(session) as B:
        session.paged_store(c.ids(B), B(k), B(v))
    assert session.device_errors() == 0
    for got, exp in zip((c.k, c.v, c.lengths), want):
        assert ref.same_bits(got, exp)


@pytest.mark.parametrize("offsets", [None, [0, 40, 80]])
def test_store_reports_what_does_not_fit(session, offsets):
    c = ref.Cache([48, 30], 1, 64, 16, F16, max_pages=3)
    grow_table(c)
    c.table[1, 2] = 10 ** 6                                # sequence 1 has no third page
    n = 80 if offsets else 2
    if not offsets:
        c.lens[1] = 33
        c.lengths.copy_(i32(c.lens))
    rows = torch.randn(n, 128, device="cuda").to(F16)
    w = torch.full((2, 1, c.slots), 5.0, device="cuda")
    p = torch.full((2, 1, c.slots), -5, dtype=torch.int32, device="cuda")
    seen = c.lengths.clone()
    want = expect_store(c, rows, 0, 64, offsets, 2, w, p, seen)
    with ref.Buffers(session) as B:
        r = B(rows)
        session.paged_store(c.ids(B), r, r, v_col=64, offsets=B(i32(offsets)) if offsets else 0, weights=B(w),
                            positions=B(p), seen=B(seen))
    assert session.device_errors() == ERR_BAD
    for got, exp in zip((c.k, c.v, c.lengths, w, p, seen), want):
        assert ref.same_bits(got, exp)


@pytest.mark.parametrize("offsets", [[5, 3, 9], [-4, 2, 100], [0, 0, 0], [9, 9, 9]])
def test_store_with_odd_offsets_stays_inside(session, offsets):
    """Offsets that are not in order, or reach past the rows, write held rows only and nothing out of place."""
    c = ref.Cache([10, 31], 1, 64, 16, BF16, max_pages=4)
    grow_table(c)
    before = c.k.clone()
    rows = torch.ones(9, 128, device="cuda").to(BF16)
    with ref.Buffers(session) as B:
        r = B(rows)
        session.paged_store(c.ids(B), r, r, v_col=64, offsets=B(i32(offsets)))
    session.device_errors()
    assert bool((c.lengths >= i32([10, 31])).all()) and bool((c.lengths <= i32([19, 40])).all())
    for b, n in enumerate([10, 31]):
        for s in range(n):
            page = int(c.table[b, s // 16])
            assert ref.same_bits(c.k[page, :, s % 16], before[page, :, s % 16])


# ------------------------------------------------------------------ eviction

def run_evict(session, c, budget, recent, w, p, seen, out=None, errors=0):
    size = capi.paged_evict_workspace_bytes(len(c.lens), c.H, c.slots, budget)
    with ref.Buffers(session) as B:
        new = dict(zip(("new_lengths", "new_weights", "new_positions"), [B(t) for t in out])) if out else {}
        session.paged_evict(c.ids(B), budget, recent, B(w), B(p), B(seen), workspace=B.workspace(size), **new)
    assert session.device_errors() == errors


def check_evict(c, budget, recent, w, p, seen, before, now):
    k, v, ow, op = before
    nk, nv, nw, npos, nlen = now
    ek, ev, ew, ep = k.clone(), v.clone(), nw.cpu().clone(), npos.cpu().clone()
    hw, hp, table = w.cpu(), p.cpu(), c.table.cpu()
    for b, n in enumerate(c.lens):
        assert int(nlen[b]) == min(n, budget)
        for h in range(c.H):
            stay, moves = ref.evict(hw[b, h].numpy(), hp[b, h].numpy(), n, budget, recent, int(seen[b]))
            to = torch.tensor(stay + [t for _, t in moves], dtype=torch.long)
            at = torch.tensor(stay + [a for a, _ in moves], dtype=torch.long)
            ew[b, h, :min(n, budget)] = 0
            ew[b, h, to], ep[b, h, to] = hw[b, h, at], hp[b, h, at]
            to, at = to[len(stay):], at[len(stay):]
            pa, pt = table[b, at // c.P].long(), table[b, to // c.P].long()
            ek[pt, h, to % c.P], ev[pt, h, to % c.P] = k[pa, h, at % c.P], v[pa, h, at % c.P]
            for got, old in ((nw, ow), (npos, op)):          # behind the new length nothing is written
                assert ref.same_bits(got[b, h, min(n, budget):], old[b, h, min(n, budget):])
    assert ref.same_bits(nk, ek) and ref.same_bits(nv, ev)
    assert np.array_equal(nw.cpu().numpy(), ew.numpy(), equal_nan=True) and torch.equal(npos.cpu(), ep)


def weights_for(kind, B, H, slots, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(2 * torch.randn(B, H, slots, generator=g))
    if kind == "ties":
        w = torch.randint(0, 3, (B, H, slots), generator=g).float()
    elif kind == "equal":
        w = torch.full((B, H, slots), 0.25)
    elif kind == "odd":
        vals = torch.tensor([math.nan, -math.nan, math.inf, -math.inf, 0.0, -0.0, -1.5, 1e-45, -1e-45, 3.0])
        w = vals[torch.randint(0, len(vals), (B, H, slots), generator=g)]
    elif kind == "close":
        w = torch.from_numpy((np.random.RandomState(seed).randint(0, 300, (B, H, slots)) + 0x3f800000)
                             .astype(np.uint32).view(np.float32))
    return w


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd", "close"])
@pytest.mark.parametrize("dtype,D,H,page,lens,budget,recent,shuffled", [
    (BF16, 64, 2, 16, [0, 1, 99, 100, 101, 180], 100, 10, False),
    (F16, 128, 1, 8, [65, 64, 2], 1, 1, False),
    (BF16, 64, 3, 32, [300, 257, 1000], 256, 256, True),
    (BF16, 256, 2, 64, [130], 77, 0, True),
    (BF16, 64, 40, 8, [536, 530, 513, 512, 30, 0], 512, 40, True),   # at most 32 moves, heads in turns
    (F16, 64, 40, 8, [700, 600, 301], 300, 0, False),
    (F16, 128, 5, 8, [1016, 1001, 1000], 1000, 5, True),
    (BF16, 64, 40, 16, [5000, 1, 4097], 4000, 100, False),
    (F16, 64, 1, 128, [3000, 2999, 0], 900, 33, True)])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict(session, kind, dtype, D, H, page, lens, budget, recent, shuffled, in_place):
    c = ref.Cache(lens, H, D, page, dtype, max_pages=-(-max(lens) // page) + 1)
    B = len(lens)
    w = weights_for(kind, B, H, c.slots).cuda()
    g = torch.Generator().manual_seed(7)
    p = torch.full((B, H, c.slots), 10 ** 6, dtype=torch.int32)
    for b, n in enumerate(lens):
        for h in range(H):
            p[b, h, :n] = torch.randperm(n, generator=g).int() if shuffled else torch.arange(n, dtype=torch.int32)
    p, seen = p.cuda(), c.lengths.clone()
    mark = (torch.full_like(w, 123.0), torch.full_like(p, -9))
    before = (c.k.cpu().clone(), c.v.cpu().clone(), *((w.clone(), p.clone()) if in_place else mark))
    w0, p0 = w.clone(), p.clone()
    if in_place:
        run_evict(session, c, budget, recent, w, p, seen)
        now = (c.k, c.v, w, p, c.lengths)
    else:
        out = (torch.full_like(c.lengths, -1), *[t.clone() for t in mark])
        run_evict(session, c, budget, recent, w, p, seen, out)
        now = (c.k, c.v, out[1], out[2], out[0])
        assert ref.same_bits(w, w0) and ref.same_bits(p, p0) and c.lengths.tolist() == lens
    check_evict(c, budget, recent, w0, p0, seen, before, now)


@pytest.mark.parametrize("n,budget", [(40001, 39999), (40001, 5000), (33000, 17), (8193, 8192), (1025, 1000),
                                      (140001, 139990), (140001, 6000),
                                      (400001, 399000), (400001, 70000)])   # the last two do not fit shared memory
def test_evict_long(session, n, budget):
    c = ref.Cache([n, n // 2], 1, 64, 64, BF16)
    w = weights_for("spread", 2, 1, c.slots, seed=n).cuda()
    w[torch.rand(w.shape, device="cuda") < 0.3] = 0.0
    p = torch.arange(c.slots, dtype=torch.int32, device="cuda").repeat(2, 1, 1)
    before = (c.k.cpu().clone(), c.v.cpu().clone(), w.clone(), p.clone())
    w0, p0 = w.clone(), p.clone()
    run_evict(session, c, budget, min(budget, 128), w, p, c.lengths.clone())
    check_evict(c, budget, min(budget, 128), w0, p0, i32(c.lens), before, (c.k, c.v, w, p, c.lengths))


@pytest.mark.parametrize("D,H,page,heads,most,budget", [
    (64, 8, 16, 320, 1500, 700), (128, 4, 32, 320, 1500, 700), (256, 2, 8, 160, 1500, 700),
    (64, 4, 64, 300, 5200, 2400)])       # many moves a head
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_of_large_batches(session, D, H, page, heads, most, budget, in_place):
    """More heads than the GPU has SMs; some sequences need no cut."""
    B = heads // H
    lens = torch.randint(most // 3, most, (B,), generator=torch.Generator().manual_seed(H)).tolist()
    lens[0], lens[-1] = 0, most
    c = ref.Cache(lens, H, D, page, BF16)
    w = weights_for("spread", B, H, c.slots, seed=H).cuda()
    w[torch.rand(w.shape, device="cuda") < 0.2] = 0.5
    p = torch.arange(c.slots, dtype=torch.int32, device="cuda").repeat(B, H, 1)
    w0, p0 = w.clone(), p.clone()
    mark = (torch.full_like(w, 123.0), torch.full_like(p, -9))
    before = (c.k.cpu().clone(), c.v.cpu().clone(), *((w0, p0) if in_place else mark))
    out = None if in_place else (torch.full_like(c.lengths, -1), *[t.clone() for t in mark])
    run_evict(session, c, budget, 60, w, p, i32(lens), out)
    now = (c.k, c.v, w, p, c.lengths) if in_place else (c.k, c.v, out[1], out[2], out[0])
    check_evict(c, budget, 60, w0, p0, i32(lens), before, now)


@pytest.mark.parametrize("n", [262144, 300000])   # in shared memory, and not
def test_evict_of_the_older_half(session, n):
    """Every slot of the recent half moves: whole rounds of 32768 slots."""
    c = ref.Cache([n], 1, 64, 64, BF16)
    w = weights_for("spread", 1, 1, c.slots, seed=n).cuda()
    p = torch.arange(c.slots, dtype=torch.int32, device="cuda").repeat(1, 1, 1)
    before = (c.k.cpu().clone(), c.v.cpu().clone(), w.clone(), p.clone())
    w0, p0 = w.clone(), p.clone()
    run_evict(session, c, n // 2, n // 2, w, p, c.lengths.clone())
    check_evict(c, n // 2, n // 2, w0, p0, i32(c.lens), before, (c.k, c.v, w, p, c.lengths))


@pytest.mark.parametrize("n", [900, 5003])
def test_evict_arrays_at_odd_addresses(session, n):
    """Weights and positions that start 4 bytes behind a 16-byte boundary."""
    c = ref.Cache([n, n - 7], 2, 64, 32, F16)
    w0 = weights_for("ties", 2, 2, c.slots).cuda()
    p0 = torch.arange(c.slots, dtype=torch.int32, device="cuda").repeat(2, 2, 1)
    before = (c.k.cpu().clone(), c.v.cpu().clone(), w0.clone(), p0.clone())
    room = [torch.empty(w0.numel() + 1, dtype=t, device="cuda") for t in (torch.float32, torch.int32)]
    w, p = (r[1:].view(w0.shape) for r in room)
    w.copy_(w0), p.copy_(p0)
    run_evict(session, c, n // 2, 50, w, p, c.lengths.clone())
    check_evict(c, n // 2, 50, w0, p0, i32(c.lens), before, (c.k, c.v, w, p, c.lengths))


def test_more_recent_slots_than_the_budget(session):
    """Positions that claim to be recent everywhere: the lowest slots are kept."""
    c = ref.Cache([50], 1, 64, 16, BF16)
    w = torch.rand(1, 1, c.slots, device="cuda")
    p = torch.full((1, 1, c.slots), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    k = c.k.clone()
    run_evict(session, c, 20, 5, w, p, i32([-2 ** 31]))
    assert ref.same_bits(c.k, k) and c.lengths.tolist() == [20]


def test_evict_reports_bad_pages(session):
    c = ref.Cache([64, 64], 1, 64, 16, BF16)
    w = torch.zeros(2, 1, c.slots, device="cuda")
    w[0, 0, 40] = w[1, 0, 40] = 1.0
    p = torch.arange(c.slots, dtype=torch.int32, device="cuda").repeat(2, 1, 1)
    c.table[1, 2] = -1
    k = c.k.clone()
    run_evict(session, c, 10, 0, w, p, i32([64, 64]), errors=ERR_BAD)
    moved = c.table[0, 0].item()
    assert ref.same_bits(c.k[moved, 0, 9], k[c.table[0, 2].item(), 0, 8])
    k[moved, 0, 9] = c.k[moved, 0, 9]
    assert ref.same_bits(c.k, k) and float(w[1, 0, 9]) == 1.0 and c.lengths.tolist() == [10, 10]


# ------------------------------------------------------------------ together

def test_decode_with_a_bounded_cache(session):
    """A run as a server makes it: prompts of several lengths enter the cache, then steps of rotary positions,
    store, attention with weights and eviction, each compared with its restatement on the inputs it had."""
    B, H, group, D, page, budget, recent = 3, 2, 3, 64, 16, 40, 8
    heads, width, slots = H * group, (H * group + 2 * H) * 64, 64
    g = torch.Generator().manual_seed(11)
    c = ref.Cache([0, 0, 0], H, D, page, BF16, max_pages=slots // page)
    grow_table(c)
    w = torch.zeros(B, H, slots, device="cuda")
    p = torch.zeros(B, H, slots, dtype=torch.int32, device="cuda")
    seen = torch.zeros(B, dtype=torch.int32, device="cuda")
    out = torch.zeros(B, heads * D, dtype=BF16, device="cuda")
    lse = torch.zeros(B, heads, device="cuda")
    prompts = torch.randn(50, width, generator=g).to(BF16).cuda()
    offsets = [0, 20, 21, 50]
    step = torch.zeros(B, width, dtype=BF16, device="cuda")
    with ref.Buffers(session) as R:
        ids, bw, bp, bs = c.ids(R), R(w), R(p), R(seen)
        where = torch.cat([torch.arange(b - a) for a, b in zip(offsets, offsets[1:])]).int().cuda()
        pr, st, bo, bl = R(prompts), R(step), R(out), R(lse)
        session.rotary(pr, pr, R(where), heads + H, D)
        ws = R.workspace(max(capi.paged_attention_workspace_bytes(B, heads, H, D, slots, True),
                             capi.paged_evict_workspace_bytes(B, H, slots, budget)))
        torch.cuda.synchronize()
        want = expect_store(c, prompts, heads * D, (heads + H) * D, offsets, B, w, p, seen)
        session.paged_store(ids, pr, pr, k_col=heads * D, v_col=(heads + H) * D, offsets=R(i32(offsets)), weights=bw,
                            positions=bp, seen=bs)
        for got, exp in zip((c.k, c.v, c.lengths, w, p, seen), want):
            assert ref.same_bits(got, exp)
        for n in range(24):
            x = torch.randn(B, width, generator=g).to(BF16)
            step.copy_(x)
            session.rotary(st, st, bs, heads + H, D)       # a new token's position is the count of those before it
            c.lens = c.lengths.tolist()
            y, far = ref.rotary(x[:, :(heads + H) * D], seen.cpu()[:, None], heads + H, D, [32], D, 1e4, False, False,
                                False)
            got = step.cpu()[:, :(heads + H) * D].double().view_as(y)
            assert bool(((got - y).abs() <= ref.half_step(y, BF16) + 2.0 ** -19 * x.abs().max()).all())
            want = expect_store(c, step, heads * D, (heads + H) * D, None, B, w, p, seen)
            session.paged_store(ids, st, st, k_col=heads * D, v_col=(heads + H) * D, weights=bw, positions=bp, seen=bs)
            for a, e in zip((c.k, c.v, c.lengths, w, p, seen), want):
                assert ref.same_bits(a, e)
            c.lens = c.lengths.tolist()
            old = w.cpu().double()
            session.paged_attention(ids, st, bo, heads, workspace=ws, lse=bl, weights=bw)
            torch.cuda.synchronize()
            sums = check(c, step[:, :heads * D].contiguous(), heads, out, lse)
            for (b, h), (s, rel) in sums.items():
                m = c.lens[b]
                total = old[b, h, :m] + s
                assert bool(((w[b, h, :m].cpu().double() - total).abs() <= s * rel + total * 2.0 ** -23).all())
            before = (c.k.cpu().clone(), c.v.cpu().clone(), w.clone(), p.clone())
            w0, p0 = w.clone(), p.clone()
            session.paged_evict(ids, budget, recent, bw, bp, bs, workspace=ws)
            torch.cuda.synchronize()
            check_evict(c, budget, recent, w0, p0, seen, before, (c.k, c.v, w, p, c.lengths))
        assert c.lengths.tolist() == [40, 25, 40] and seen.tolist() == [44, 25, 53]
        for b in range(B):                                 # every head still holds the latest tokens, once each
            for h in range(H):
                held = sorted(p[b, h, :c.lengths[b]].tolist())
                assert len(set(held)) == len(held) and held[-recent:] == list(range(int(seen[b]) - recent, int(seen[b])))
    assert session.device_errors() == 0


def views(c):
    return capi.fer_paged_view_t(c.k.data_ptr(), c.v.data_ptr(), c.table.data_ptr(), c.lengths.data_ptr(),
                                 len(c.lens), c.max_pages, c.k.shape[0], c.H, c.P, c.D, ref.CODES[c.dtype])


def test_captured_steps(session):
    """The launchers in two graphs with a workspace each, replayed at once on two streams, against eager calls."""
    lib = capi.kernels()
    runs, err = [], torch.zeros(1, dtype=torch.int32, device="cuda")
    for seed in (0, 1):
        c = ref.Cache([90, 200, 0, 31], 2, 64, 16, BF16, max_pages=20, seed=seed)
        grow_table(c)
        B, heads = 4, 4
        t = dict(rows=torch.randn(B, 8 * 64, device="cuda").to(BF16), out=torch.zeros(B, heads * 64, dtype=BF16, device="cuda"),
                 w=torch.zeros(B, 2, c.slots, device="cuda"),
                 p=torch.arange(c.slots, dtype=torch.int32, device="cuda").repeat(B, 2, 1), seen=c.lengths.clone(),
                 lse=torch.zeros(B, heads, device="cuda"))
        size = max(lib.fer_paged_attention_workspace_bytes(B, heads, 2, 64, c.slots, 1),
                   lib.fer_paged_evict_workspace_bytes(B, 2, c.slots, 60))
        t["ws"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        runs.append((c, t, size))

    def step(c, t, size, stream):
        v, e = views(c), err.data_ptr()
        a = capi.fer_rotary_args_t(t["rows"].data_ptr(), t["rows"].data_ptr(), t["seen"].data_ptr(), 512, 512, 4, 6, 64,
                                   64, 1, (C.c_int * 4)(32), 1e4, 0, capi.FER_DTYPE_BF16)
        assert lib.fer_rotary(C.byref(a), stream) == 0
        s = capi.fer_paged_store_args_t(t["rows"].data_ptr() + 512, t["rows"].data_ptr() + 768, 512, 512, 4, 4, None,
                                        c.lengths.data_ptr(), t["w"].data_ptr(), t["p"].data_ptr(),
                                        t["seen"].data_ptr(), t["seen"].data_ptr())
        assert lib.fer_paged_store(C.byref(v), C.byref(s), e, stream) == 0
        q = capi.fer_paged_attention_args_t(t["rows"].data_ptr(), t["out"].data_ptr(), 512, 256, 4, 4, 0.0,
                                            t["lse"].data_ptr(), t["w"].data_ptr(), t["ws"].data_ptr(), size)
        assert lib.fer_paged_attention(C.byref(v), C.byref(q), e, stream) == 0
        x = capi.fer_paged_evict_args_t(60, 9, t["w"].data_ptr(), t["p"].data_ptr(), t["seen"].data_ptr(),
                                        c.lengths.data_ptr(), t["w"].data_ptr(), t["p"].data_ptr(),
                                        t["ws"].data_ptr(), size)
        assert lib.fer_paged_evict(C.byref(v), C.byref(x), e, stream) == 0

    state = [{k: x.clone() for k, x in dict(t, k=c.k, v=c.v, lengths=c.lengths).items()} for c, t, _ in runs]
    eager = []
    for c, t, size in runs:
        for _ in range(5):
            step(c, t, size, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        eager.append([x.clone() for x in (c.k, c.v, c.lengths, t["w"], t["p"], t["seen"], t["out"], t["lse"])])
    for (c, t, _), s in zip(runs, state):
        for k, x in dict(t, k=c.k, v=c.v, lengths=c.lengths).items():
            x.copy_(s[k])
    graphs, streams = [], [torch.cuda.Stream() for _ in runs]
    for (c, t, size), st in zip(runs, streams):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            step(c, t, size, torch.cuda.current_stream().cuda_stream)
        graphs.append(gr)
    torch.cuda.synchronize()
    for _ in range(5):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for (c, t, _), want in zip(runs, eager):
        for got, exp in zip((c.k, c.v, c.lengths, t["w"], t["p"], t["seen"], t["out"], t["lse"]), want):
            assert ref.same_bits(got, exp)
    assert int(err) == 0


@pytest.mark.parametrize("lens,H,budget", [([5000, 3000, 20], 2, 1000), ([1500] * 160, 2, 700)])
def test_captured_long_eviction(lens, H, budget):
    """Selection in clusters, and with the moves in the same kernel, replayed from a graph in place."""
    lib = capi.kernels()
    c = ref.Cache(lens, H, 64, 64, BF16)
    B, err = len(lens), torch.zeros(1, dtype=torch.int32, device="cuda")
    w = weights_for("spread", B, H, c.slots).cuda()
    p = torch.arange(c.slots, dtype=torch.int32, device="cuda").repeat(B, H, 1)
    seen = c.lengths.clone()
    size = lib.fer_paged_evict_workspace_bytes(B, H, c.slots, budget)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    v = views(c)
    a = capi.fer_paged_evict_args_t(budget, 50, w.data_ptr(), p.data_ptr(), seen.data_ptr(), c.lengths.data_ptr(),
                                    w.data_ptr(), p.data_ptr(), ws.data_ptr(), size)
    state = (c.k, c.v, w, p, c.lengths)
    before = [x.clone() for x in state]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert lib.fer_paged_evict(C.byref(v), C.byref(a), err.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    for _ in range(2):
        for x, old in zip(state, before):
            x.copy_(old)
        graph.replay()
        torch.cuda.synchronize()
        check_evict(c, budget, 50, before[2], before[3], seen, [before[0].cpu(), before[1].cpu(), *before[2:4]], state)
    assert int(err) == 0


FIRST_USE = """
import ctypes as C, sys
sys.path.insert(0, {root!r})
import torch
from fercuda_b200 import capi
from tests import paged_ref as ref
lib = capi.kernels()
c = ref.Cache([90, 300], 2, {dim}, 16, torch.bfloat16, max_pages=30)
W = 2 * {dim}
q = torch.randn(2, W, device="cuda").to(torch.bfloat16)
out = torch.zeros_like(q)
w, p = torch.zeros(2, 2, c.slots, device="cuda"), torch.zeros(2, 2, c.slots, dtype=torch.int32, device="cuda")
seen = c.lengths.clone()
size = max(lib.fer_paged_attention_workspace_bytes(2, 2, 2, {dim}, c.slots, 1), lib.fer_paged_evict_workspace_bytes(2, 2, c.slots, 60))
ws = torch.empty(size, dtype=torch.uint8, device="cuda")
v = capi.fer_paged_view_t(c.k.data_ptr(), c.v.data_ptr(), c.table.data_ptr(), c.lengths.data_ptr(), 2, c.max_pages,
                          c.k.shape[0], 2, 16, {dim}, capi.FER_DTYPE_BF16)
a = capi.fer_rotary_args_t(q.data_ptr(), q.data_ptr(), seen.data_ptr(), W, W, 2, 2, {dim}, {dim}, 1, (C.c_int * 4)({dim} // 2),
                           1e4, 0, capi.FER_DTYPE_BF16)
x = capi.fer_paged_attention_args_t(q.data_ptr(), out.data_ptr(), W, W, 2, 2, 0.0, None, w.data_ptr(), ws.data_ptr(), size)
e = capi.fer_paged_evict_args_t(60, 9, w.data_ptr(), p.data_ptr(), seen.data_ptr(), c.lengths.data_ptr(), w.data_ptr(),
                                p.data_ptr(), ws.data_ptr(), size)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    s = torch.cuda.current_stream().cuda_stream
    rc = [lib.fer_rotary(C.byref(a), s), lib.fer_paged_attention(C.byref(v), C.byref(x), None, s),
          lib.fer_paged_evict(C.byref(v), C.byref(e), None, s)]
assert rc == [0, 0, 0], rc
g.replay()
torch.cuda.synchronize()
print("ok", c.lengths.tolist(), float(out.float().abs().sum()) > 0)
"""


@pytest.mark.parametrize("dim", [64, 128])
def test_first_use_under_capture(dim):
    """A process whose first calls of the launchers are captured."""
    root = str(Path(__file__).resolve().parents[1])
    r = subprocess.run([sys.executable, "-c", FIRST_USE.format(root=root, dim=dim)], capture_output=True, text=True,
                       timeout=240, cwd=root)
    assert r.returncode == 0 and "ok [60, 60] True" in r.stdout, r.stdout + r.stderr


def test_session_calls_are_refused_under_capture(session):
    c = ref.Cache([20], 1, 64, 16, BF16)
    q, out = queries(c, 1), torch.zeros(1, 64, dtype=BF16, device="cuda")
    st = torch.cuda.Stream()
    with ref.Buffers(session) as B:
        ids, bq, bo = c.ids(B), B(q), B(out)
        ws = B.workspace(capi.paged_attention_workspace_bytes(1, 1, 1, 64, c.slots))
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            session.set_stream(torch.cuda.current_stream().cuda_stream)
            with pytest.raises(capi.FerError) as e:
                session.paged_attention(ids, bq, bo, 1, workspace=ws)
            out.add_(1)
        assert "captured" in e.value.msg
        session.set_stream(torch.cuda.current_stream().cuda_stream)
        session.wait(session.paged_attention(ids, bq, bo, 1, workspace=ws))
    check(c, q, 1, out, attend(session, c, q, 1)[1])


def test_another_stream(session):
    """Work queued on a side stream, behind a copy on that stream that brings the query."""
    c = ref.Cache([3000] * 4, 4, 128, 16, BF16)
    q = queries(c, 4)
    want, _ = attend(session, c, q, 4)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        late, out = torch.zeros_like(q), torch.zeros_like(q)
        with ref.Buffers(session) as B:
            ws = B.workspace(capi.paged_attention_workspace_bytes(4, 4, 4, 128, c.slots))
            big = torch.ones(1 << 27, device="cuda")
            for _ in range(5):
                big.mul_(1.0001)
            late.copy_(q)
            job = session.paged_attention(c.ids(B), B(late), B(out), 4, workspace=ws)
            session.wait(job)
    assert ref.same_bits(out, want)


def make(session_bufs, **change):
    """Arguments of the three calls on a small cache, some of them replaced."""
    c = ref.Cache([20, 5], 2, 64, 16, BF16, max_pages=3)
    grow_table(c)
    t = dict(k=c.k, v=c.v, table=c.table, lengths=c.lengths, q=torch.zeros(2, 256, dtype=BF16, device="cuda"),
             out=torch.zeros(2, 256, dtype=BF16, device="cuda"), w=torch.zeros(2, 2, 48, device="cuda"),
             p=torch.zeros(2, 2, 48, dtype=torch.int32, device="cuda"), seen=c.lengths.clone(),
             lse=torch.zeros(2, 4, device="cuda"), ws=torch.zeros(1 << 20, dtype=torch.uint8, device="cuda"),
             off=i32([0, 1, 2]), rows=torch.zeros(2, 256, dtype=BF16, device="cuda"), new=c.lengths.clone())
    t.update({k: f(t) for k, f in change.items()})
    return {k: session_bufs(x) for k, x in t.items()}


BAD_CACHE = [dict(k=lambda t: t["k"].float()), dict(v=lambda t: t["v"].to(F16)), dict(v=lambda t: t["v"][:-1].clone()),
             dict(k=lambda t: t["k"].view(-1, 2, 16 * 64)), dict(table=lambda t: t["table"].float()),
             dict(table=lambda t: t["table"].view(-1)), dict(lengths=lambda t: i32([1, 2, 3])),
             dict(v=lambda t: t["k"]), dict(lengths=lambda t: t["table"].view(-1)[:2]),
             dict(k=lambda t: t["k"].view(-1, 2, 32, 32), v=lambda t: t["v"].view(-1, 2, 32, 32)),
             dict(k=lambda t: t["k"].view(-1, 8, 4, 64), v=lambda t: t["v"].view(-1, 8, 4, 64))]
BAD_ATTENTION = [dict(q=lambda t: t["q"].to(F16)), dict(out=lambda t: t["out"].float()), dict(out=lambda t: t["q"]),
                 dict(q=lambda t: t["q"][:, :128].clone()), dict(out=lambda t: t["out"][:1].clone()),
                 dict(q=lambda t: t["q"].repeat(2, 1), out=lambda t: t["out"].repeat(2, 1)),
                 dict(lse=lambda t: t["lse"].view(-1)), dict(w=lambda t: t["w"][:, :, :47].clone()),
                 dict(w=lambda t: t["p"].clone()), dict(ws=lambda t: t["ws"][:100].clone()),
                 dict(ws=lambda t: t["ws"][4:]), dict(ws=lambda t: t["w"].view(-1)),
                 dict(lse=lambda t: t["w"].view(-1)[:8].view(2, 4)), dict(out=lambda t: t["k"].view(-1, 256)[:2])]
BAD_STORE = [dict(rows=lambda t: t["rows"].to(F16)), dict(rows=lambda t: t["rows"][:, :128].clone()),
             dict(rows=lambda t: t["rows"].repeat(2, 1), off=lambda t: None), dict(off=lambda t: i32([0])),
             dict(off=lambda t: i32([0, 1, 2, 2])), dict(off=lambda t: t["off"].float()),
             dict(seen=lambda t: None), dict(seen=lambda t: i32([1])), dict(new=lambda t: t["seen"]),
             dict(new=lambda t: i32([1])), dict(rows=lambda t: t["k"].view(-1, 256)[:2]),
             dict(p=lambda t: t["w"]), dict(w=lambda t: t["p"].view(torch.float32))]
BAD_EVICT = [dict(w=lambda t: t["w"][:1].clone()), dict(p=lambda t: t["p"].float()), dict(seen=lambda t: i32([1])),
             dict(new=lambda t: t["seen"]), dict(ws=lambda t: t["ws"][:4].clone()),
             dict(ws=lambda t: t["p"].view(torch.uint8).view(-1)), dict(new=lambda t: t["table"].view(-1)[:2])]


def refused(fn):
    with pytest.raises(capi.FerError) as e:
        fn()
    assert e.value.code == capi.FER_STATUS_INVALID_ARGUMENT


def calls(session, t):
    cache = capi.paged_cache(t["k"], t["v"], t["table"], t["lengths"])
    return (lambda **kw: session.paged_attention(cache, t["q"], t["out"], kw.pop("heads", 4), workspace=t["ws"],
                                                 lse=t["lse"], weights=t["w"], **kw),
            lambda **kw: session.paged_store(cache, t["rows"], t["rows"], **{**dict(
                v_col=128, offsets=t["off"], new_lengths=t["new"], weights=t["w"], positions=t["p"],
                seen=t["seen"]), **kw}),
            lambda **kw: session.paged_evict(cache, kw.pop("budget", 10), kw.pop("recent", 2), t["w"], t["p"],
                                             t["seen"], workspace=t["ws"], new_lengths=t["new"], **kw))


@pytest.mark.parametrize("change", BAD_CACHE)
def test_cache_refusals(session, change):
    with ref.Buffers(session) as B:
        for fn in calls(session, make(B, **change)):
            refused(fn)


@pytest.mark.parametrize("which,change", [(0, x) for x in BAD_ATTENTION] + [(1, x) for x in BAD_STORE] +
                         [(2, x) for x in BAD_EVICT])
def test_refusals(session, which, change):
    with ref.Buffers(session) as B:
        refused(calls(session, make(B, **change))[which])


@pytest.mark.parametrize("which,kw", [
    (0, dict(heads=0)), (0, dict(heads=3)), (0, dict(heads=6)), (0, dict(q_col=1)), (0, dict(out_col=1)),
    (0, dict(scale=-1.0)), (0, dict(scale=math.nan)), (1, dict(k_col=129)), (1, dict(v_col=129)),
    (1, dict(seen=0)), (2, dict(budget=0)), (2, dict(recent=11))])
def test_argument_refusals(session, which, kw):
    with ref.Buffers(session) as B:
        refused(lambda: calls(session, make(B))[which](**kw))


def test_unknown_buffers(session):
    with ref.Buffers(session) as B:
        t = make(B)
        for which, names in ((0, ("k", "table", "q", "out", "ws", "lse", "w")), (1, ("v", "rows", "off", "new", "p")),
                             (2, ("lengths", "w", "p", "seen", "ws", "new"))):
            for n in names:
                with pytest.raises(capi.FerError) as e:
                    calls(session, dict(t, **{n: 10 ** 9}))[which]()
                assert e.value.code == capi.FER_STATUS_NOT_FOUND, n
        for fn in calls(session, t):                       # and as made they are taken
            fn()
    assert session.device_errors() == 0
