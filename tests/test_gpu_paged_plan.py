"""fer_submit_paged_plan against a loop over the sequences, one page at a time: all numbers are exact."""
import ctypes as C

import pytest
import torch

from fercuda_b200 import capi
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

ERR_BAD = 4


def plan(table, lengths, counts, held, seen, ring, state, page, rows):
    """(table, ring, new_held, new_state, offsets, sequences, positions, slots, bad)."""
    table, ring = [list(r) for r in table], list(ring)
    pages, per, bad = len(ring), len(table[0]), False
    first, free = state
    broken = not (0 <= first < pages and 0 <= free <= pages)
    if broken:
        bad, room = True, 0
        first, free = 0, 0
    else:
        room = pages - free
    new_held, offsets, put, asked, takes = [], [0], [], 0, 0
    seqs, poss, slots = [], [], []
    for b, (n, c, h) in enumerate(zip(lengths, counts, held)):
        if not 0 <= n <= per * page or c < 0 or not 0 <= h <= per:
            bad = True
        n, c, h = min(max(n, 0), per * page), max(c, 0), min(max(h, 0), per)
        if n + c > per * page:
            bad, c = True, 0
        need, keep = -(-(n + c) // page), -(-n // page)
        ask = max(need - h, 0)
        asked += ask
        on = ask == 0 or asked <= free
        after = h if broken else need if on else min(h, keep)
        if on:
            for j in range(h, after):
                table[b][j] = ring[(first + takes) % pages]
                bad |= not 0 <= table[b][j] < pages
                takes += 1
        for j in range(after, h):
            if len(put) < room:
                bad |= not 0 <= table[b][j] < pages
                put.append(table[b][j])
            else:
                bad = True
        new_held.append(after)
        count = c if on else 0
        offsets.append(offsets[-1] + count)
        for i in range(count):
            s = n + i
            seqs.append(b), poss.append((n if seen is None else seen[b]) + i)
            p = table[b][s // page]
            good = 0 <= p < pages
            if rows is None or len(slots) < rows:
                bad |= not good
            slots.append(p * page + s % page if good else -1)
    for i, p in enumerate(put):
        ring[(first + free + i) % pages] = p
    state = list(state) if broken else [(first + takes) % pages, free - takes + len(put)]
    if rows is None:
        rows = len(seqs)
    bad |= offsets[-1] > rows
    pad = max(0, rows - len(seqs))
    return table, ring, new_held, state, offsets, (seqs + [-1] * pad)[:rows], (poss + [0] * pad)[:rows], (slots + [-1] * pad)[:rows], bad


def make(batch, page, per, seed, spare=None, most=None, ended=0.1, running=0.6):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))  # noqa: E731
    pages = batch * per + 5
    order = torch.randperm(pages, generator=g).tolist()
    table, lengths, counts, held, seen = [], [], [], [], []
    cap, at = per * page, 0
    kinds = torch.rand(batch, generator=g).tolist()
    for b in range(batch):
        if kinds[b] < ended:
            n, c, h = 0, 0, rnd(0, per)
        elif kinds[b] < ended + running:
            n = rnd(1, cap - 1)
            c, h = 1, -(-n // page) + (1 if rnd(0, 9) == 0 else 0)
        else:
            n, c, h = 0, rnd(0, min(cap, most or cap)), 0
        h = min(h, per)
        table.append(order[at:at + h] + [-9] * (per - h))
        at += h
        lengths.append(n), counts.append(c), held.append(h), seen.append(n + rnd(0, 5))
    free = pages - at if spare is None else min(spare, pages - at)
    first = rnd(0, pages - 1)
    ring = [-8] * pages
    for i in range(free):
        ring[(first + i) % pages] = order[at + i]
    return table, lengths, counts, held, seen, ring, [first, free]


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def check(session, table, lengths, counts, held, seen, ring, state, page, rows, in_place=False, arrays=(1, 1, 1)):
    want = plan(table, lengths, counts, held, seen, ring, state, page, rows if any(arrays) else None)
    t = dict(table=i32(table), ring=i32(ring), held=i32(held), state=i32(state), offsets=i32([7] * (len(lengths) + 1)))
    t["new_held"], t["new_state"] = (t["held"], t["state"]) if in_place else (i32([7] * len(lengths)), i32([7, 7]))
    row = [i32([7] * rows) if a else None for a in arrays]
    with ref.Buffers(session) as B:
        b = {k: B(v) for k, v in t.items() if k not in ("new_held", "new_state") or not in_place}
        session.paged_plan(b["table"], B(i32(lengths)), B(i32(counts)), b["held"], b["ring"], b["state"], b["offsets"], page_size=page,
                           new_held=b.get("new_held", 0), new_free_state=b.get("new_state", 0), sequences=B(row[0]),
                           positions=B(row[1]), slots=B(row[2]), seen=B(None if seen is None else i32(seen)))
    bad = want[-1]
    assert session.device_errors() == (ERR_BAD if bad else 0)
    got = (t["table"], t["ring"], t["new_held"], t["new_state"], t["offsets"], *row)
    for name, a, w in zip(("table", "ring", "held", "state", "offsets", "sequences", "positions", "slots"), got, want):
        if a is not None:
            assert a.cpu().tolist() == w, name
    if not in_place:
        assert t["held"].cpu().tolist() == list(held) and t["state"].cpu().tolist() == list(state)
    return want


# few rows: one small CTA; up to 4096: one; up to 16384: a cluster; more: a launch of their own
@pytest.mark.parametrize("batch,page,per,most,tail", [
    (1, 16, 4, None, 0), (1, 8, 1, None, 3), (7, 8, 5, 20, 5), (64, 16, 12, 10, 7), (256, 32, 4, 2, 1),
    (257, 16, 6, 4, 0), (200, 64, 9, 90, 3), (100, 256, 4, 900, 1), (300, 16, 40, 500, 9), (200, 256, 4, 1000, 6), (1500, 8, 6, 30, 2), (5000, 16, 3, 3, 2),
    (9000, 8, 2, 5, 11)])
@pytest.mark.parametrize("tight", [False, True])
def test_matches_a_loop(session, batch, page, per, most, tail, tight):
    a = make(batch, page, per, batch + page, spare=batch * per // 12 if tight else None, most=most)
    total = plan(*a, page, None)[4][-1]
    check(session, *a, page, total + tail + (total == 0), in_place=bool(batch % 2))


@pytest.mark.parametrize("arrays", [(0, 0, 0), (1, 0, 0), (0, 1, 0), (0, 0, 1)])
@pytest.mark.parametrize("batch", [5, 400])
def test_arrays_that_are_left_out(session, arrays, batch):
    a = list(make(batch, 16, 5, 4, most=30))
    rows = plan(*a, 16, None)[4][-1] + 2
    check(session, *a, 16, rows, arrays=arrays)
    a[4] = None
    check(session, *a, 16, rows, arrays=arrays)


@pytest.mark.parametrize("batch", [6, 300, 2000])
def test_more_rows_than_the_arrays_have(session, batch):
    a = make(batch, 16, 5, 11, most=30)
    total = plan(*a, 16, None)[4][-1]
    for rows in (1, total // 2 + 1, total - 1):
        assert check(session, *a, 16, rows)[-1]


@pytest.mark.parametrize("state", [[-1, 3], [10 ** 6, 3], [0, -1], [0, 10 ** 6], [2 ** 31 - 1, 2 ** 31 - 1]])
@pytest.mark.parametrize("batch", [5, 400])
def test_a_broken_ring_moves_no_page(session, state, batch):
    a = list(make(batch, 16, 5, 5, most=30))
    table, held = a[0], a[3]
    a[6] = state
    want = check(session, *a, 16, 50)
    assert want[0] == table and want[2] == held and want[-1]


@pytest.mark.parametrize("batch", [12, 600])
def test_bad_numbers_are_clamped_and_reported(session, batch):
    for which, values in ((1, (-1, 2 ** 31 - 1, -2 ** 31, 81)), (2, (-5, 2 ** 31 - 1, 80)), (3, (-1, 6, 2 ** 31 - 1))):
        for v in values:
            a = [list(x) for x in make(batch, 16, 5, 6, most=30)]
            if which == 3 and v > 5:     # pages of the row, all of them real
                a[0][2] = [0, 1, 2, 3, 4]
            a[which][2] = v
            if which == 1:
                a[3][2] = 0
            check(session, *a, 16, 40 * batch)


@pytest.mark.parametrize("batch", [12, 600])
def test_bad_page_ids_are_reported(session, batch):
    a = make(batch, 16, 5, 7, most=30)
    b = next(i for i in range(batch) if a[1][i] and a[3][i])
    a[0][b][a[3][b] - 1] = 10 ** 9
    a[2][b] = 1
    a[1][b] = a[3][b] * 16 - 1     # its new row is in the bad page
    assert check(session, *a, 16, 40 * batch)[-1]
    a = make(batch, 16, 5, 7, most=30)
    a[5][a[6][0]] = -4             # the first free page
    a[2][0], a[1][0], a[3][0], a[0][0] = 20, 0, 0, [-9] * 5
    assert check(session, *a, 16, 40 * batch)[-1]


def test_pages_for_which_the_ring_has_no_room(session):
    """More pages than there are: some belong to two."""
    a = [list(x) for x in make(5, 16, 4, 3)]
    n = len(a[5])
    a[6] = [3, n - 2]
    a[5] = list(range(n))
    a[1], a[2], a[3] = [0] * 5, [0] * 5, [4, 0, 0, 2, 0]
    a[0][0], a[0][3] = [1, 2, 3, 4], [5, 6, -9, -9]
    want = check(session, *a, 16, 4)
    assert want[-1] and want[3] == [3, n]


def test_steps_go_round_the_ring(session):
    """Forty steps in place: requests enter, grow and end; no page is ever in two places."""
    page, per, batch = 8, 6, 40
    table, lengths, counts, held, seen, ring, state = make(batch, page, per, 21, spare=60, ended=0.0, running=0.0, most=20)
    g = torch.Generator().manual_seed(2)
    every = sorted(ring[(state[0] + i) % len(ring)] for i in range(state[1]))
    for step in range(40):
        want = check(session, table, lengths, counts, held, None, ring, state, page, 400, in_place=bool(step % 2))
        table, ring, held, state, offsets = want[:5]
        owned = [p for b in range(batch) for p in table[b][:held[b]]]
        owned += [ring[(state[0] + i) % len(ring)] for i in range(state[1])]
        assert sorted(owned) == every
        lengths = [n + offsets[b + 1] - offsets[b] for b, n in enumerate(lengths)]
        over = torch.rand(batch, generator=g).tolist()
        fresh = torch.randint(0, 25, (batch,), generator=g).tolist()
        counts = [0] * batch
        for b in range(batch):
            if lengths[b] == 0:
                counts[b] = fresh[b]
            elif over[b] < 0.15 or lengths[b] >= per * page - 1:
                lengths[b] = 0      # ended: its pages go back in the next step
            else:
                counts[b] = 1


def test_captured_and_replayed_in_place(session):
    page, per, batch, rows = 16, 4, 30, 100
    table, lengths, counts, held, seen, ring, state = make(batch, page, per, 31, most=3)
    t = [i32(v) for v in (table, lengths, counts, held, seen, ring, state)]
    off, row = i32([0] * (batch + 1)), [i32([7] * rows) for _ in range(3)]
    a = capi.fer_paged_plan_args_t(t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), t[3].data_ptr(), t[4].data_ptr(), t[5].data_ptr(),
                                   t[6].data_ptr(), t[3].data_ptr(), t[6].data_ptr(), off.data_ptr(), *(r.data_ptr() for r in row),
                                   batch, per, len(ring), page, rows)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert capi.kernels().fer_paged_plan(C.byref(a), None, torch.cuda.current_stream().cuda_stream) == 0
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
        want = plan(table, lengths, counts, held, seen, ring, state, page, rows)
        table, ring, held, state = want[:4]
        for got, w in zip((t[0], t[5], t[3], t[6], off, *row), want):
            assert got.cpu().tolist() == w
        lengths = [n + want[4][b + 1] - want[4][b] for b, n in enumerate(lengths)]
        counts = [1 if 0 < n < per * page else 0 for n in lengths]
        lengths[3] = counts[3] = 0
        t[1].copy_(i32(lengths)), t[2].copy_(i32(counts))
    del graph


@pytest.mark.parametrize("change,word", [
    (dict(table="ring"), "page table"), (dict(lengths="ring"), "[batch]"), (dict(counts="f32"), "[batch]"), (dict(held="short"), "[batch]"),
    (dict(seen="short"), "[batch]"), (dict(ring="table"), "free_pages"), (dict(state="held"), "free_state"),
    (dict(new_state="held"), "free_state"), (dict(offsets="held"), "offsets"), (dict(sequences="f32"), "rows"),
    (dict(slots="more"), "rows"), (dict(page=24), "page_size"), (dict(page=4), "page_size"), (dict(page=512), "page_size"),
    (dict(new_held="lengths"), "overlap"), (dict(sequences="positions"), "overlap"), (dict(new_state="in_ring"), "overlap")])
def test_refusals(session, change, word):
    table, lengths, counts, held, seen, ring, state = make(3, 16, 4, 1)
    dev = i32(ring)
    with ref.Buffers(session) as B:
        bufs = dict(table=B(i32(table)), lengths=B(i32(lengths)), counts=B(i32(counts)), held=B(i32(held)), seen=B(i32(seen)),
                    ring=B(dev), state=B(i32(state)), new_held=B(i32(held)), new_state=B(i32(state)), offsets=B(i32([0] * 4)),
                    sequences=B(i32([0] * 9)), positions=B(i32([0] * 9)), slots=B(i32([0] * 9)), more=B(i32([0] * 10)),
                    short=B(i32([0] * 2)), f32=B(torch.zeros(9, device="cuda")),
                    in_ring=session.import_ptr(capi.FER_DTYPE_I32, [2], dev.data_ptr()))
        B.ids.append(bufs["in_ring"])
        p = lambda n: bufs[change.get(n, n)]  # noqa: E731
        with pytest.raises(capi.FerError) as e:
            session.paged_plan(p("table"), p("lengths"), p("counts"), p("held"), p("ring"), p("state"), p("offsets"),
                               page_size=change.get("page", 16), new_held=p("new_held"), new_free_state=p("new_state"),
                               sequences=p("sequences"), positions=p("positions"), slots=p("slots"), seen=p("seen"))
    assert e.value.code == capi.FER_STATUS_INVALID_ARGUMENT and word in e.value.msg, e.value.msg
