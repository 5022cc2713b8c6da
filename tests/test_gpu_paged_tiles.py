"""Windowed attention of prompts and single tokens over a paged cache, and
attention behind a shared prefix, against 64-bit restatements (tests/tiles_ref.py,
where the bounds are derived). Pages are NaN outside the held slots, and table
entries behind them are no page ids, so anything that is read there shows."""
import ctypes as C
import math

import pytest
import torch

from fercuda_b200 import capi
from tests import paged_ref as ref
from tests import tiles_ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
ERR_BAD = 4
MARK = 7.0


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def queries(rows, width, dtype, seed=1, factor=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, width, generator=g) * factor).to(dtype).cuda()


def window(session, c, q, heads, offsets, win, sinks, *, q_col=0, out=None, out_col=0, scale=0.0, errors=0, rows=None):
    rows = q.shape[0]
    out = torch.full((rows, heads * c.D), MARK, dtype=c.dtype, device="cuda") if out is None else out
    lse = torch.full((rows, heads), MARK, device="cuda")
    seqs = rows if offsets is None else len(offsets) - 1
    with ref.Buffers(session) as B:
        size = capi.paged_window_attention_workspace_bytes(rows, seqs, heads, c.H, c.D, c.slots, win, sinks)
        bq = B(q)
        session.paged_window_attention(c.ids(B), bq, bq if out is q else B(out), heads, win, sinks,
                                       offsets=B(i32(offsets)) if offsets is not None else 0, lse=B(lse),
                                       workspace=B.workspace(size), q_col=q_col, out_col=out_col, scale=scale)
    assert session.device_errors() == errors
    return out, lse


def agree(got, glse, want, wlse, err, ds, dtype):
    got, glse = got.cpu().double().view_as(want), glse.cpu().double()
    mine = ~want[..., 0].isnan()
    assert torch.equal(got[~mine], torch.full_like(got[~mine], MARK)) and bool((glse[~mine] == MARK).all())
    off = (got - want).abs()[mine]
    assert bool((off <= (ref.half_step(want, dtype) + err)[mine]).all()), float(off.max())
    some = wlse > -math.inf
    assert torch.equal(glse[mine] > -math.inf, some[mine])
    assert bool(((glse - wlse)[mine & some].abs() <= ds + wlse[mine & some].abs() * 2.0 ** -21 + 2.0 ** -20).all())


def check_window(session, c, q, heads, offsets, win, sinks, scale=None, skip=(), errors=0, **kw):
    out, lse = window(session, c, q, heads, offsets, win, sinks, scale=scale or 0.0, errors=errors, **kw)
    agree(out, lse, *tiles_ref.window(c, q, heads, offsets, win, sinks, scale, skip), c.dtype)
    return out, lse


# one token a sequence: no, short, ragged and long windows, sinks that meet the window, empty places
@pytest.mark.parametrize("dtype,D,H,group,page,lens,win,sinks", [
    (BF16, 64, 1, 1, 8, [1], 0, 0),
    (BF16, 64, 2, 1, 16, [0, 1, 2, 127, 128, 129], 0, 0),
    (F16, 128, 2, 4, 16, [300, 0, 64, 65, 7], 64, 4),
    (BF16, 128, 1, 16, 8, [513, 512, 1000], 1, 0),
    (BF16, 256, 2, 3, 64, [200, 63, 0, 129], 100, 130),
    (F16, 256, 1, 40, 256, [600], 77, 1),          # rows of several kinds of units: 40 of 128
    (BF16, 128, 1, 140, 32, [300, 10], 200, 8),    # more than a sub-tile's rows
    (F16, 64, 1, 300, 128, [260], 0, 0),           # more than a unit's
    (BF16, 64, 4, 5, 32, [1500, 1300], 1200, 3),   # parts that are joined
    (F16, 128, 1, 2, 64, [5000], 0, 0),
    (BF16, 128, 1, 2, 64, [3000], 10 ** 9, 2 * 10 ** 9),
])
def test_window_of_single_tokens(session, dtype, D, H, group, page, lens, win, sinks):
    c = ref.Cache(lens, H, D, page, dtype, seed=D + len(lens))
    check_window(session, c, queries(len(lens), H * group * D, dtype), H * group, None, win, sinks)


# sinks in chunks of their own, or meeting the window's; windows that begin inside a page; more units than CTAs; no slot or page
# outside is any number
@pytest.mark.parametrize("dtype,D,H,group,page,lens,win,sinks", [
    (BF16, 64, 2, 4, 256, [2000, 1500, 700, 257], 100, 600),
    (F16, 128, 2, 8, 8, [3000, 1290, 1300, 20], 1000, 300),
    (BF16, 128, 1, 9, 128, [1000, 999, 64, 65], 64, 1),
    (BF16, 256, 2, 16, 16, [1200, 130, 0, 513], 300, 64),
    (F16, 64, 16, 1, 16, [(i * 37) % 900 for i in range(70)], 200, 5),
    (BF16, 128, 8, 4, 64, [(i * 211) % 2000 for i in range(40)], 1024, 4),
    (BF16, 128, 2, 17, 16, [1200, 130, 700], 300, 64),
    (F16, 64, 1, 2, 8, [70000, 66000, 3], 66000, 3),      # longer chunks
])
def test_window_of_single_tokens_reads_nothing_else(session, dtype, D, H, group, page, lens, win, sinks):
    c = ref.Cache(lens, H, D, page, dtype, seed=win)
    q = queries(len(lens), H * group * D, dtype)
    dev, k, v, table = (c.k, c.v, c.table), c.k.cpu(), c.v.cpu(), c.table.cpu()
    c.k, c.v, c.table = k, v, table      # read over and over
    want = tiles_ref.window(c, q, H * group, None, win, sinks)
    c.k, c.v, c.table = dev
    for b, n in enumerate(lens):
        gone = torch.arange(n)
        gone = gone[(gone >= sinks) & (gone <= n - 1 - win)]
        at = table[b, gone // page].long()
        k[at, :, gone % page], v[at, :, gone % page] = math.nan, math.inf
        for i in (gone // page).unique().tolist():
            if i * page >= sinks and (i + 1) * page <= n - win:
                table[b, i] = [-1, 10 ** 9, -2 ** 31][i % 3]
    c.k.copy_(k), c.v.copy_(v), c.table.copy_(table)
    out, lse = window(session, c, q, H * group, None, win, sinks)
    agree(out, lse, *want, dtype)
    if lens[0] > win:      # a page that is read is reported
        c.table[0, (lens[0] - 1) // page] = -1
        window(session, c, q, H * group, None, win, sinks, errors=ERR_BAD)


# prompts: ragged rows, sequences without any, rows behind the last, more rows than slots
@pytest.mark.parametrize("dtype,D,H,group,page,lens,new,win,sinks,tail", [
    (BF16, 64, 2, 1, 16, [5], [5], 0, 0, 0),
    (BF16, 128, 2, 4, 16, [64, 200, 0, 33], [64, 70, 0, 1], 0, 0, 3),
    (F16, 128, 1, 8, 8, [300, 129], [130, 129], 50, 4, 1),
    (BF16, 256, 1, 2, 64, [150, 90], [100, 90], 33, 5, 0),
    (F16, 64, 1, 3, 32, [260, 1, 40], [200, 1, 40], 1, 0, 2),
    (BF16, 128, 1, 1, 128, [600], [400], 150, 70, 0),
    (BF16, 64, 1, 4, 256, [700], [90], 0, 0, 0),
    (F16, 128, 2, 2, 16, [20, 50], [30, 10], 0, 0, 0),      # the first 10 rows of one sequence have no slot
    (BF16, 128, 1, 7, 64, [9000], [40], 0, 0, 0),           # few rows over many keys: joined parts
    (F16, 256, 1, 5, 16, [5000], [60], 3000, 9, 4),
])
def test_window_of_prompts(session, dtype, D, H, group, page, lens, new, win, sinks, tail):
    c = ref.Cache(lens, H, D, page, dtype, seed=D + sum(new))
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    check_window(session, c, queries(offsets[-1] + tail, H * group * D, dtype), H * group, offsets, win, sinks)


def test_window_of_fewer_sequences_than_the_cache_has(session):
    c = ref.Cache([70, 30, 90], 2, 64, 16, BF16)
    q = queries(40, 4 * 64, BF16)
    out, lse = window(session, c, q, 4, [0, 25, 38], 20, 2)
    c.lens = c.lens[:2]
    agree(out, lse, *tiles_ref.window(c, q, 4, [0, 25, 38], 20, 2), BF16)


@pytest.mark.parametrize("scale", [1e-3, 0.7, 3.0])
def test_window_scale(session, scale):
    c = ref.Cache([90, 41], 1, 64, 16, F16)
    check_window(session, c, queries(50, 2 * 64, F16, factor=1.0), 2, [0, 30, 41], 0, 0, scale=scale)


@pytest.mark.parametrize("q_col,out_col,group,offsets", [
    (0, 512, 4, None), (3, 517, 4, None), (8, 520, 3, [0, 2, 9]), (1, 601, 5, [0, 4, 9]), (16, 700, 4, [0, 9, 9])])
def test_window_columns_of_a_fused_activation(session, q_col, out_col, group, offsets):
    """Queries and results as columns of one buffer, at odd places too; the other columns stay as they are."""
    c = ref.Cache([150, 9], 1, 64, 16, BF16)
    rows, width = (2 if offsets is None else 9), group * 64
    fused = queries(rows, 1040, BF16)
    before = fused.clone()
    window(session, c, fused, group, offsets, 40, 3, q_col=q_col, out=fused, out_col=out_col)
    q = before[:, q_col: q_col + width].contiguous()
    want, _, err, _ = tiles_ref.window(c, q, group, offsets, 40, 3)
    got = fused[:, out_col: out_col + width].cpu().double().view_as(want)
    mine = ~want[..., 0].isnan()
    assert bool(((got - want).abs() <= ref.half_step(want, BF16) + err)[mine].all())
    rest = torch.ones(1040, dtype=torch.bool)
    rest[out_col: out_col + width] = False
    assert torch.equal(fused.cpu()[:, rest], before.cpu()[:, rest])


def poison(c, b, h, slots, k=None, v=None):
    for s in slots:
        p = int(c.table[b, s // c.P])
        if k is not None:
            c.k[p, h, s % c.P] = k
        if v is not None:
            c.v[p, h, s % c.P] = v


@pytest.mark.parametrize("D,new", [(64, None), (128, [100]), (256, [100]), (128, [3])])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see_does_not_matter(session, D, new, bad):
    """Infinities and NaN before the window, behind the prompt's rows, and among rows that others see."""
    n = 300
    c = ref.Cache([n], 2, D, 16, BF16, max_pages=24)
    offsets = None if new is None else [0, new[0]]
    rows = 1 if new is None else new[0]
    q = queries(rows, 4 * D, BF16)
    win, sinks = 60, 3
    clean = window(session, c, q, 4, offsets, win, sinks)
    first = n - rows
    poison(c, 0, 0, range(sinks, first + 1 - win), bad, bad)            # seen by no row
    out, lse = window(session, c, q, 4, offsets, win, sinks)
    assert ref.same_bits(out, clean[0]) and ref.same_bits(lse, clean[1])
    if rows > 60:
        # seen by the later rows only, and by the earlier ones only
        poison(c, 0, 1, [n - 20], None, bad)
        poison(c, 0, 1, [first - 30], None, bad)
        out, lse = window(session, c, q, 4, offsets, win, sinks)
        got, was = out.view(rows, 4, D), clean[0].view(rows, 4, D)
        at = torch.arange(first, n)
        sees = ((at >= n - 20) | (at - win < first - 30)).cuda()
        assert torch.equal(got[:, :2], was[:, :2])
        assert torch.equal(got[~sees][:, 2:], was[~sees][:, 2:])
        wrong = got[sees][:, 2:]
        assert bool((wrong.isnan() if math.isnan(bad) else wrong == bad).all())
        assert ref.same_bits(lse, clean[1])


def test_scores_of_lowest_and_infinite_values(session):
    """Scores of -inf count as nothing; rows whose scores are all -inf give zeros."""
    c = ref.Cache([70, 40], 1, 64, 16, F16)
    c.k.nan_to_num_(0.0), c.v.nan_to_num_(0.0)
    q = torch.ones(2, 64, dtype=F16, device="cuda")
    poison(c, 0, 0, range(0, 69), -math.inf)
    poison(c, 1, 0, range(0, 40), -math.inf)
    out, lse = window(session, c, q, 1, None, 0, 0)
    v = c.rows(c.v, 0, 0)[69]
    assert bool(((out[0].cpu().double() - v).abs() <= ref.half_step(v, F16)).all())
    assert bool((out[1] == 0).all()) and lse[1].item() == -math.inf and math.isfinite(lse[0].item())
    poison(c, 0, 0, range(0, 69), -65504.0)
    out, _ = window(session, c, q, 1, None, 0, 0)
    assert bool(((out[0].cpu().double() - v).abs() <= ref.half_step(v, F16)).all())


@pytest.mark.parametrize("D,group,new", [(64, 4, 70), (128, 4, 70), (256, 4, 70), (128, 2, 50), (64, 3, 5), (256, 2, 1), (128, 1, None)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_scores_of_infinity_and_nan(session, D, group, new, bad):
    """They make the rows that see them NaN, wherever they stand, and no other."""
    n = 300
    rows, offsets = (1, None) if new is None else (new, [0, new])
    q = queries(rows, group * D, BF16).abs()
    for at in (*range(n - 19, n), 0, 5, 130, n - 40):
        c = ref.Cache([n], 1, D, 16, BF16)
        poison(c, 0, 0, [at], k=torch.tensor([bad] + [1.0] * (D - 1), dtype=BF16, device="cuda"))
        sees = torch.arange(n - rows, n) >= at
        for win in (0, 200):
            out, lse = window(session, c, q, group, offsets, win, 1)
            see = sees & (torch.arange(n - rows, n) - win < at) if win and at else sees
            got = out.view(rows, group, D).cpu()
            assert bool(got[see].isnan().all()) and bool(lse.cpu()[see].isnan().all())
            assert bool(got[~see].isfinite().all()) and bool(lse.cpu()[~see].isfinite().all())


def test_prefix_scores_of_infinity_and_nan(session):
    for bad in (math.nan, math.inf):
        c = Shared(300, [20] * 40, 1, 128, 16, BF16)
        q = queries(40, 4 * 128, BF16).abs()
        p = int(c.table[3, 0])
        c.k[p, 0, 8, 5] = bad
        out, lse = prefix(session, c, c.prefix, 300, q, 4)
        see = torch.arange(40) == 3
        assert bool(out.cpu()[see].isnan().all()) and bool(lse.cpu()[see].isnan().all())
        assert bool(out.cpu()[~see].isfinite().all()) and bool(lse.cpu()[~see].isfinite().all())
        c.k[c.prefix[9], 0, 0, 5] = bad
        out, lse = prefix(session, c, c.prefix, 300, q, 4)
        assert bool(out.isnan().all()) and bool(lse.isnan().all())


def test_rows_without_slots_behind_a_long_window(session):
    """Rows before slot 0 and a window near 2^31."""
    c = ref.Cache([20, 50], 2, 64, 16, F16)
    q = queries(300, 4 * 64, F16)
    offsets = [0, 200, 300]
    want = window(session, c, q, 4, offsets, 0, 0)
    for win in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 100):
        got = check_window(session, c, q, 4, offsets, win, 3)
        assert ref.same_bits(got[0], want[0]) and ref.same_bits(got[1], want[1])


def test_growing_scores(session):
    """Every block's maximum is far above the one before, and far below at the end."""
    c = ref.Cache([1400], 1, 128, 64, BF16)
    for s0 in range(0, 1400, 64):
        size = float(min(s0, 1400 - s0)) / 40
        poison(c, 0, 0, range(s0, min(s0 + 64, 1400)), torch.full((128,), size, dtype=BF16, device="cuda"))
    q = torch.ones(300, 2 * 128, dtype=BF16, device="cuda")
    check_window(session, c, q, 2, [0, 300], 0, 0)
    check_window(session, c, q, 2, [0, 300], 500, 4)


def test_pages_outside_every_window_are_not_read(session):
    """Their entries may be anything, and so may their rows."""
    c = ref.Cache([400, 350], 2, 128, 16, F16)
    q = queries(60, 4 * 128, F16)
    offsets = [0, 40, 60]
    want = window(session, c, q, 4, offsets, 50, 5)
    for b, n in ((0, 400 - 40), (1, 350 - 20)):
        gone = range(1, (n + 1 - 50) // 16)
        for i in gone:
            p = int(c.table[b, i])
            c.k[p], c.v[p] = math.nan, math.nan
            c.table[b, i] = [-1, 10 ** 9, 2 ** 31 - 1][i % 3]
    out, lse = window(session, c, q, 4, offsets, 50, 5)
    assert ref.same_bits(out, want[0]) and ref.same_bits(lse, want[1])


@pytest.mark.parametrize("D,lens,new", [(128, [200, 90], None), (128, [200, 90], [150, 40]), (256, [200, 90], [30, 2]), (64, [600, 90], [1, 1])])
def test_bad_pages_and_lengths_are_reported(session, D, lens, new):
    c = ref.Cache(lens, 1, D, 16, BF16, max_pages=40)
    offsets = None if new is None else [0, new[0], sum(new)]
    rows = 2 if new is None else sum(new)
    q = queries(rows, 2 * D, BF16)
    c.table[0, 3] = c.k.shape[0]
    c.table[1, 0] = -5
    c.lengths[:] = i32(lens)
    # a page is looked up where a row of a tile sees a slot of it: the rows of the reference see the same slots or fewer
    skip = [(0, s) for s in range(48, 64)] + [(1, s) for s in range(16)]
    keep = c.table.clone()
    c.table[0, 3], c.table[1, 0] = 0, 0        # for the restatement's own reading
    want = tiles_ref.window(c, q, 2, offsets, 0, 0, None, skip)
    c.table.copy_(keep)
    out, lse = window(session, c, q, 2, offsets, 0, 0, errors=ERR_BAD)
    agree(out, lse, *want, BF16)
    c.table[0, 3], c.table[1, 0] = 0, 0
    c.lengths[0] = 10 ** 6
    window(session, c, q, 2, offsets, 0, 0, errors=ERR_BAD)
    c.lengths[0] = -1
    window(session, c, q, 2, offsets, 0, 0, errors=ERR_BAD)


@pytest.mark.parametrize("offsets", [[0, 9, 5], [-1, 3, 5], [0, 2, 99], [5, 3, 1], [2 ** 31 - 1, 0, 4], [0, 10, 0]])
def test_bad_offsets_are_reported(session, offsets):
    c = ref.Cache([20, 20], 1, 64, 16, F16)
    window(session, c, queries(10, 2 * 64, F16), 2, offsets, 0, 0, errors=ERR_BAD)


def test_the_same_bits_every_time(session):
    c = ref.Cache([3000, 77, 0, 1234], 2, 128, 16, BF16)
    q = queries(200, 8 * 128, BF16)
    offsets = [0, 150, 160, 160, 200]
    first = window(session, c, q, 8, offsets, 900, 4)
    for _ in range(3):
        again = window(session, c, q, 8, offsets, 900, 4)
        assert ref.same_bits(first[0], again[0]) and ref.same_bits(first[1], again[1])


def test_many_short_sequences(session):
    """More sequences than the table of units has entries, some without rows."""
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 40, (700,), generator=g).tolist()
    new = [min(n, int(i % 4)) for i, n in enumerate(lens)]
    c = ref.Cache(lens, 1, 64, 8, F16)
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    check_window(session, c, queries(offsets[-1] + 2, 2 * 64, F16), 2, offsets, 9, 2)
    check_window(session, c, queries(700, 2 * 64, F16), 2, None, 0, 0)


def test_elements_behind_two_to_the_31(session):
    """Pages whose elements lie behind 2^31 of a pool."""
    pages, H, P, D = 9000, 8, 256, 128          # 2.36 G elements
    k = torch.zeros(pages, H, P, D, dtype=BF16, device="cuda")
    v = torch.zeros_like(k)
    c = ref.Cache([300], H, D, P, BF16)
    for i, p in enumerate((pages - 1, pages - 3)):
        k[p], v[p] = c.k[int(c.table[0, i])], c.v[int(c.table[0, i])]
    want = window(session, c, queries(20, H * D, BF16), H, [0, 20], 0, 0)
    c.k, c.v = k, v
    c.table[0, :2] = i32([pages - 1, pages - 3])
    got = window(session, c, queries(20, H * D, BF16), H, [0, 20], 0, 0)
    assert ref.same_bits(got[0], want[0])
    del k, v, c
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ a shared prefix

def prefix(session, c, pages, length, q, heads, *, scale=0.0, errors=0):
    out = torch.full((q.shape[0], heads * c.D), MARK, dtype=c.dtype, device="cuda")
    lse = torch.full((q.shape[0], heads), MARK, device="cuda")
    with ref.Buffers(session) as B:
        size = capi.paged_prefix_attention_workspace_bytes(q.shape[0], heads, c.H, c.D, c.slots, len(pages) * c.P)
        session.paged_prefix_attention(c.ids(B), B(i32(pages)), B(i32([length])), B(q), B(out), heads, lse=B(lse),
                                       workspace=B.workspace(size), scale=scale)
    assert session.device_errors() == errors
    return out, lse


class Shared(ref.Cache):
    """A cache whose pools also hold a prefix of `length` slots, in pages of its own."""

    def __init__(self, length, lens, H, D, page, dtype, width=None, **kw):
        need = -(-length // page)
        super().__init__([length] + list(lens), H, D, page, dtype, **kw)
        self.prefix = self.table[0, :need].tolist() + [-3] * ((width or need) - need)
        self.lens, self.table, self.lengths = self.lens[1:], self.table[1:].contiguous(), self.lengths[1:].contiguous()


@pytest.mark.parametrize("dtype,D,H,group,page,length,lens", [
    (BF16, 64, 1, 1, 16, 1, [1]),
    (BF16, 64, 2, 4, 16, 100, [5, 0, 31, 200]),
    (F16, 128, 2, 4, 16, 700, [40, 0, 300, 129, 1]),
    (BF16, 128, 1, 8, 64, 2049, [7] * 40),              # rows of two sub-tiles
    (F16, 64, 1, 3, 8, 333, [20] * 100),                # a group that does not divide a tile
    (BF16, 256, 1, 5, 32, 515, [64, 65, 0] * 10),
    (F16, 128, 3, 1, 256, 1000, [700, 2, 0]),
    (BF16, 128, 1, 300, 16, 140, [20, 3]),
    # sequences enough that their own slots are the other kernel's work: one chunk, several, none
    (BF16, 128, 8, 4, 16, 700, [(i * 53) % 300 for i in range(40)]),
    (F16, 64, 32, 1, 8, 300, [600, 0, 257, 256, 1, 511, 512, 513, 30, 800]),
    (BF16, 256, 6, 2, 64, 130, [(i * 7) % 70 for i in range(50)]),
    (F16, 128, 150, 16, 32, 200, [400, 33]),
    (F16, 128, 150, 17, 32, 200, [40, 33]),
    (BF16, 64, 300, 2, 16, 50, [0]),
])
def test_prefix(session, dtype, D, H, group, page, length, lens):
    c = Shared(length, lens, H, D, page, dtype, width=-(-length // page) + 2, seed=length)
    q = queries(len(lens), H * group * D, dtype)
    out, lse = prefix(session, c, c.prefix, length, q, H * group)
    agree(out, lse, *tiles_ref.prefix(c, c.prefix, length, q, H * group), dtype)


def test_prefix_of_nothing(session):
    """No prefix at all, and sequences that hold nothing either."""
    c = Shared(16, [30, 0], 1, 64, 16, F16)
    q = queries(2, 2 * 64, F16)
    out, lse = prefix(session, c, c.prefix, 0, q, 2)
    agree(out, lse, *tiles_ref.prefix(c, c.prefix, 0, q, 2), F16)
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())


def test_prefix_own_pages_out_of_range(session):
    """Of many sequences: reported, and of no weight."""
    c = Shared(100, [40] * 50, 6, 64, 16, BF16)
    q = queries(50, 12 * 64, BF16)
    c.table[7, 1] = -1
    out, lse = prefix(session, c, c.prefix, 100, q, 12, errors=ERR_BAD)
    c.table[7, 1] = 0
    others = torch.arange(50) != 7
    want, wlse, err, ds = tiles_ref.prefix(c, c.prefix, 100, q, 12)
    agree(out.view(50, 12, 64)[others], lse[others], want[others], wlse[others], err[others], ds, BF16)
    assert bool(out.isfinite().all())
    c.lengths[9] = -3
    prefix(session, c, c.prefix, 100, q, 12, errors=ERR_BAD)


def test_prefix_the_same_bits_every_time(session):
    c = Shared(3000, [(i * 97) % 900 for i in range(64)], 8, 128, 16, F16)
    q = queries(64, 32 * 128, F16)
    first = prefix(session, c, c.prefix, 3000, q, 32)
    for _ in range(3):
        again = prefix(session, c, c.prefix, 3000, q, 32)
        assert ref.same_bits(first[0], again[0]) and ref.same_bits(first[1], again[1])


def test_prefix_captured_and_replayed(session):
    """With another prefix, other lengths and other pages in each replay."""
    c = Shared(700, [200] * 40, 8, 128, 16, BF16)
    q = queries(40, 32 * 128, BF16)
    out, lse = torch.zeros(40, 32 * 128, dtype=BF16, device="cuda"), torch.zeros(40, 32, device="cuda")
    pages, length = i32(c.prefix), i32([700])
    ws = torch.full((capi.paged_prefix_attention_workspace_bytes(40, 32, 8, 128, c.slots, len(c.prefix) * 16),), 255,
                    dtype=torch.uint8, device="cuda")
    v, a = views(c), capi.fer_paged_prefix_args_t(q.data_ptr(), out.data_ptr(), 32 * 128, 32 * 128, 40, 32, pages.data_ptr(),
                                                  length.data_ptr(), len(c.prefix), 0.0, lse.data_ptr(), ws.data_ptr(), ws.numel())
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert capi.kernels().fer_paged_prefix_attention(C.byref(v), C.byref(a), err.data_ptr(),
                                                         torch.cuda.current_stream().cuda_stream) == 0
    for n, lens in ((700, [200] * 40), (33, [(i * 31) % 200 for i in range(40)]), (0, [i % 3 for i in range(40)])):
        length.copy_(i32([n])), c.lengths.copy_(i32(lens))
        pages.copy_(i32(c.prefix[::-1] if n == 33 else c.prefix))
        if n == 33:   # the last page of the text is its only part full
            pages[0], pages[-1] = pages[-1].clone(), pages[0].clone()
        graph.replay()
        torch.cuda.synchronize()
        c.lens = lens
        agree(out, lse, *tiles_ref.prefix(c, pages.tolist(), n, q, 32), BF16)
    assert err.item() == 0
    del graph


def test_prefix_is_what_attention_over_a_joined_table_gives(session):
    """The same keys, once as a prefix and once as the first pages of every sequence's own table."""
    length, lens = 512, [40, 17, 130]
    c = Shared(length, lens, 2, 128, 16, BF16)
    q = queries(3, 8 * 128, BF16)
    out, lse = prefix(session, c, c.prefix, length, q, 8)
    j = ref.Cache.__new__(ref.Cache)
    j.__dict__.update(c.__dict__)
    j.table = torch.cat([i32(c.prefix).expand(3, -1), c.table], 1).contiguous()
    j.max_pages = j.table.shape[1]
    j.slots = j.max_pages * 16
    j.lens = [n + length for n in lens]
    j.lengths = i32(j.lens)
    want, wlse, err, ds = tiles_ref.window(j, q, 8, None, 0, 0)
    agree(out, lse, want, wlse, err, ds, BF16)
    two, tlse = window(session, j, q, 8, None, 0, 0)
    agree(two, tlse, want, wlse, err, ds, BF16)


def test_prefix_errors_are_reported(session):
    c = Shared(100, [20, 30], 1, 64, 16, BF16)
    q = queries(2, 2 * 64, BF16)
    good = prefix(session, c, c.prefix, 100, q, 2)
    prefix(session, c, c.prefix, 10 ** 6, q, 2, errors=ERR_BAD)
    prefix(session, c, c.prefix, -1, q, 2, errors=ERR_BAD)
    pages = list(c.prefix)
    pages[2] = 10 ** 9
    out, _ = prefix(session, c, pages, 100, q, 2, errors=ERR_BAD)
    k = torch.ones(100, dtype=torch.bool)
    k[32:48] = False
    assert bool(out.isfinite().all())
    c.table[1, 1] = -1
    prefix(session, c, c.prefix, 100, q, 2, errors=ERR_BAD)
    c.table[1, 1] = 0
    assert bool(good[0].isfinite().all())


def test_prefix_of_infinite_values(session):
    """An infinite value that everybody sees is everybody's result."""
    c = Shared(300, [20] * 40, 1, 128, 16, BF16)
    c.v[c.prefix[3], 0, 5, 7] = math.inf
    q = queries(40, 4 * 128, BF16, factor=0.1)
    out, _ = prefix(session, c, c.prefix, 300, q, 4)
    got = out.view(40, 4, 128)
    assert bool((got[..., 7] == math.inf).all()) and bool(got[..., :7].isfinite().all()) and bool(got[..., 8:].isfinite().all())


# ------------------------------------------------------------------ streams, captures, refusals

def views(c):
    return capi.fer_paged_view_t(c.k.data_ptr(), c.v.data_ptr(), c.table.data_ptr(), c.lengths.data_ptr(), c.table.shape[0],
                                 c.table.shape[1], c.k.shape[0], c.H, c.P, c.D,
                                 capi.FER_DTYPE_F16 if c.dtype == F16 else capi.FER_DTYPE_BF16)


def launch_window(c, q, out, lse, ws, heads, offsets, win, sinks, stream, err=None):
    a = capi.fer_paged_window_args_t(q.data_ptr(), out.data_ptr(), q.shape[1], out.shape[1], q.shape[0],
                                     q.shape[0] if offsets is None else offsets.shape[0] - 1, heads,
                                     None if offsets is None else offsets.data_ptr(), win, sinks, 0.0, lse.data_ptr(),
                                     ws.data_ptr(), ws.numel())
    return capi.kernels().fer_paged_window_attention(C.byref(views(c)), C.byref(a), None if err is None else err.data_ptr(),
                                                     stream)


def test_two_streams_and_a_captured_graph(session):
    """Calls on two streams at once, with a workspace each, and one captured and replayed with other lengths, rows and pages."""
    c = ref.Cache([900, 300, 60], 2, 128, 16, BF16, max_pages=80)
    q = queries(90, 8 * 128, BF16)
    off = i32([0, 60, 80, 90])
    size = capi.paged_window_attention_workspace_bytes(90, 3, 8, 2, 128, c.slots, 200, 4)
    want = window(session, c, q, 8, off.tolist(), 200, 4)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    made = [(torch.full_like(want[0], MARK), torch.full_like(want[1], MARK), torch.full((size,), 255, dtype=torch.uint8, device="cuda"))
            for _ in streams]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (o, l, w) in zip(streams, made):
            assert launch_window(c, q, o, l, w, 8, off, 200, 4, s.cuda_stream) == 0
    torch.cuda.synchronize()
    for o, l, _ in made:
        assert ref.same_bits(o, want[0]) and ref.same_bits(l, want[1])
    out, lse, ws = made[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert launch_window(c, q, out, lse, ws, 8, off, 200, 4, torch.cuda.current_stream().cuda_stream) == 0
    for lens, offsets in (([900, 300, 60], [0, 60, 80, 90]), ([700, 290, 60], [0, 10, 50, 70]), ([5, 0, 1], [0, 5, 5, 6])):
        c.lengths.copy_(i32(lens)), off.copy_(i32(offsets))
        out.fill_(MARK), lse.fill_(MARK)
        graph.replay()
        torch.cuda.synchronize()
        was, c.lens = c.lens, lens
        agree(out, lse, *tiles_ref.window(c, q, 8, offsets, 200, 4), BF16)
        c.lens = was
    del graph


def test_session_calls_are_refused_under_capture(session):
    c = Shared(40, [20], 1, 64, 16, BF16)
    q, out = queries(1, 64, BF16), torch.zeros(1, 64, dtype=BF16, device="cuda")
    with ref.Buffers(session) as B:
        ids, bq, bo, bp, bl, ws = c.ids(B), B(q), B(out), B(i32(c.prefix)), B(i32([40])), B.workspace(1 << 20)
        graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        before = session.stream()
        with torch.cuda.graph(graph, stream=s):
            session.set_stream(torch.cuda.current_stream().cuda_stream)
            out.add_(0)
            for call in (lambda: session.paged_window_attention(ids, bq, bo, 1, 0, 0, workspace=ws),
                         lambda: session.paged_prefix_attention(ids, bp, bl, bq, bo, 1, workspace=ws)):
                with pytest.raises(capi.FerError) as e:
                    call()
                assert "captured" in e.value.msg
        session.set_stream(before)
    del graph


@pytest.mark.parametrize("change,word", [
    (dict(heads=3), "multiple"), (dict(heads=0), "multiple"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"),
    (dict(q_col=1), "columns"), (dict(out_col=1), "columns"), (dict(window=2 ** 31), "window"), (dict(sinks=2 ** 31), "window"),
    (dict(out="q"), "overlap"), (dict(lse="bad"), "lse"), (dict(ws="small"), "workspace"), (dict(offsets="long"), "sequences"),
    (dict(offsets="f32"), "offsets"), (dict(q="f32"), "dtype"), (dict(lse="q"), "lse"), (dict(ws="f32"), "workspace"),
    (dict(out="k"), "same rows"), (dict(offsets="ws"), "overlap")])
def test_window_refusals(session, change, word):
    c = ref.Cache([20, 9], 2, 64, 16, BF16)
    q = queries(2, 4 * 64, BF16)
    with ref.Buffers(session) as B:
        ids = c.ids(B)
        words = torch.zeros(4096, dtype=torch.uint8, device="cuda")
        bufs = dict(q=B(q), out=B(torch.zeros_like(q)), lse=B(torch.zeros(2, 4, device="cuda")), ws=B(words),
                    bad=B(torch.zeros(2, 3, device="cuda")), small=B(torch.zeros(8, dtype=torch.uint8, device="cuda")),
                    long=B(i32([0, 1, 1, 2])), f32=B(torch.zeros(2, 4 * 64, device="cuda")), k=ids.k)
        words_at = session.import_ptr(capi.FER_DTYPE_I32, [3], words.data_ptr())
        pick = lambda n, d: bufs[change.get(n, d)] if change.get(n, d) else 0  # noqa: E731
        offsets = words_at if change.get("offsets") == "ws" else pick("offsets", None)
        with pytest.raises(capi.FerError) as e:
            session.paged_window_attention(ids, pick("q", "q"), pick("out", "out"), change.get("heads", 4),
                                           change.get("window", 5), change.get("sinks", 1), workspace=pick("ws", "ws"),
                                           offsets=offsets, lse=pick("lse", "lse"), q_col=change.get("q_col", 0),
                                           out_col=change.get("out_col", 0), scale=change.get("scale", 0.0))
        session.free(words_at)
    assert e.value.code == capi.FER_STATUS_INVALID_ARGUMENT and word in e.value.msg, e.value.msg


@pytest.mark.parametrize("change,word", [
    (dict(pages="f32"), "prefix_pages"), (dict(length="pages"), "prefix_length"), (dict(ws="small"), "workspace"),
    (dict(out="q"), "overlap"), (dict(heads=3), "multiple"), (dict(rows=5), "rows"), (dict(lse="bad"), "lse")])
def test_prefix_refusals(session, change, word):
    c = Shared(40, [20, 9], 2, 64, 16, BF16)
    q = queries(change.get("rows", 2), 4 * 64, BF16)
    with ref.Buffers(session) as B:
        bufs = dict(q=B(q), out=B(torch.zeros_like(q)), pages=B(i32(c.prefix)), length=B(i32([40])),
                    ws=B(torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")), f32=B(torch.zeros(3, device="cuda")),
                    small=B(torch.zeros(16, dtype=torch.uint8, device="cuda")), bad=B(torch.zeros(2, 3, device="cuda")))
        with pytest.raises(capi.FerError) as e:
            session.paged_prefix_attention(c.ids(B), bufs[change.get("pages", "pages")], bufs[change.get("length", "length")],
                                           bufs["q"], bufs[change.get("out", "out")], change.get("heads", 4),
                                           workspace=bufs[change.get("ws", "ws")],
                                           lse=bufs[change["lse"]] if "lse" in change else 0)
    assert e.value.code == capi.FER_STATUS_INVALID_ARGUMENT and word in e.value.msg, e.value.msg


def test_unknown_buffers(session):
    c = ref.Cache([20], 1, 64, 16, BF16)
    with ref.Buffers(session) as B:
        ids = c.ids(B)
        b = B(queries(1, 64, BF16))
        for call in (lambda: session.paged_window_attention(ids, 10 ** 9, b, 1, 0, 0, workspace=b),
                     lambda: session.paged_window_attention(ids, b, b, 1, 0, 0, workspace=b, offsets=10 ** 9),
                     lambda: session.paged_prefix_attention(ids, 10 ** 9, b, b, b, 1, workspace=b)):
            with pytest.raises(capi.FerError) as e:
                call()
            assert e.value.code == capi.FER_STATUS_NOT_FOUND
