"""A serving step made of the operators, as they are used: plan, norm and rotary
of the fused activation's q and k heads in place, store, attention of the step's
prompts and single tokens; over steps in which requests enter, grow and end, once
by a session and once as one captured graph. Every stage is held against its
definition; attention against the rows that went in, not against the pages."""
import ctypes as C
import math

import pytest
import torch

from fercuda_b200 import capi
from tests import paged_ref as ref
from tests import test_gpu_norm_rotary as nr
from tests import test_gpu_paged_plan as pl
from tests import tiles_ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
B, H, HKV, D, PAGE, PER, ROWS, WIN, SINKS = 6, 4, 2, 64, 8, 12, 130, 40, 3
W = (H + 2 * HKV) * D


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Server:
    """The tensors of a serving process: pages that are NaN until they are written."""

    def __init__(self):
        pages = B * PER // 4 + 2      # too few for everybody at once
        self.pages = pages
        g = torch.Generator().manual_seed(5)
        self.k = torch.full((pages, HKV, PAGE, D), math.nan, dtype=BF16, device="cuda")
        self.v = self.k.clone()
        self.table, self.held, self.lengths = i32([[-1] * PER] * B), i32([0] * B), i32([0] * B)
        self.ring, self.state = torch.randperm(pages, generator=g).int().cuda(), i32([4, pages])
        self.counts, self.offsets = i32([0] * B), i32([0] * (B + 1))
        self.seqs, self.positions, self.slots = (i32([0] * ROWS) for _ in range(3))
        self.x = torch.zeros(ROWS, W, dtype=BF16, device="cuda")
        self.out = torch.zeros(ROWS, H * D, dtype=BF16, device="cuda")
        self.lse = torch.zeros(ROWS, H, device="cuda")
        self.qg, self.kg = ((1 + 0.3 * torch.randn(D, generator=g)).cuda() for _ in range(2))
        size = capi.paged_window_attention_workspace_bytes(ROWS, B, H, HKV, D, PER * PAGE, WIN, SINKS)
        self.ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def by_session(self, session):
        with ref.Buffers(session) as R:
            ids = {n: R(t) for n, t in vars(self).items() if isinstance(t, torch.Tensor)}
            cache = capi.paged_cache(ids["k"], ids["v"], ids["table"], ids["lengths"])
            session.paged_plan(ids["table"], ids["lengths"], ids["counts"], ids["held"], ids["ring"], ids["state"], ids["offsets"],
                               page_size=PAGE, sequences=ids["seqs"], positions=ids["positions"], slots=ids["slots"])
            session.norm_rotary(ids["x"], ids["x"], ids["positions"], H + HKV, D, k_heads=HKV, q_gamma=ids["qg"], k_gamma=ids["kg"])
            session.paged_store(cache, ids["x"], ids["x"], k_col=H * D, v_col=(H + HKV) * D, offsets=ids["offsets"])
            session.paged_window_attention(cache, ids["x"], ids["out"], H, WIN, SINKS, offsets=ids["offsets"], lse=ids["lse"],
                                           workspace=ids["ws"])
        assert session.device_errors() == 0

    def launch(self, s):
        lib, p, e = capi.kernels(), lambda t: t.data_ptr(), self.err.data_ptr()  # noqa: E731
        a = capi.fer_paged_plan_args_t(p(self.table), p(self.lengths), p(self.counts), p(self.held), None, p(self.ring), p(self.state),
                                       p(self.held), p(self.state), p(self.offsets), p(self.seqs), p(self.positions), p(self.slots),
                                       B, PER, self.pages, PAGE, ROWS)
        n = capi.fer_norm_rotary_args_t()
        n.rotary = capi.fer_rotary_args_t(p(self.x), p(self.x), p(self.positions), W, W, ROWS, H + HKV, D, D, 1, (D // 2,), 1e4, 0,
                                          capi.FER_DTYPE_BF16)
        n.k_heads, n.q_gamma, n.k_gamma, n.eps = HKV, p(self.qg), p(self.kg), 1e-6
        view = capi.fer_paged_view_t(p(self.k), p(self.v), p(self.table), p(self.lengths), B, PER, self.pages, HKV, PAGE, D,
                                     capi.FER_DTYPE_BF16)
        x = p(self.x)
        st = capi.fer_paged_store_args_t(x + 2 * H * D, x + 2 * (H + HKV) * D, W, W, ROWS, B, p(self.offsets), p(self.lengths))
        at = capi.fer_paged_window_args_t(x, p(self.out), W, H * D, ROWS, B, H, p(self.offsets), WIN, SINKS, 0.0, p(self.lse),
                                          p(self.ws), self.ws.numel())
        assert lib.fer_paged_plan(C.byref(a), e, s) == 0
        assert lib.fer_norm_rotary(C.byref(n), e, s) == 0
        assert lib.fer_paged_store(C.byref(view), C.byref(st), e, s) == 0
        assert lib.fer_paged_window_attention(C.byref(view), C.byref(at), e, s) == 0


class Rows:
    """The held rows of every sequence as they went in, in the form tiles_ref takes."""
    H, D, dtype, k, v = HKV, D, BF16, 0, 1

    def __init__(self):
        self.held = [[] for _ in range(B)]     # (keys, values), each [HKV, D]

    @property
    def lens(self):
        return [len(h) for h in self.held]

    def rows(self, which, b, h):
        return torch.stack([kv[which][h] for kv in self.held[b]]).double() if self.held[b] else torch.zeros(0, D, dtype=torch.float64)


@pytest.mark.parametrize("captured", [False, True])
def test_serving_steps(session, captured):
    s, known = Server(), Rows()
    g = torch.Generator().manual_seed(9)
    graph = None
    if captured:
        s.launch(torch.cuda.current_stream().cuda_stream)     # counts are 0: nothing happens, and kernels are loaded
        torch.cuda.synchronize()
        assert s.state.tolist() == [4, s.pages] and s.offsets.tolist() == [0] * (B + 1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.launch(torch.cuda.current_stream().cuda_stream)
    waited = ended = 0
    for step in range(24):
        prompts = torch.randint(1, 60, (B,), generator=g).tolist()
        dice = torch.rand(B, generator=g).tolist()
        counts = [1] * B
        for b in range(B):
            if known.lens[b] and (dice[b] < 0.15 or known.lens[b] >= PER * PAGE):
                known.held[b], counts[b], ended = [], 0, ended + 1
            elif not known.lens[b]:
                counts[b] = prompts[b] if dice[b] < 0.5 else 0
        while sum(counts) > ROWS:
            counts[counts.index(max(counts))] = 1
        s.lengths.copy_(i32(known.lens)), s.counts.copy_(i32(counts))
        x = torch.randn(ROWS, W, generator=g).to(BF16)
        s.x.copy_(x)
        s.out.fill_(7.0), s.lse.fill_(7.0)
        want = pl.plan(s.table.tolist(), known.lens, counts, s.held.tolist(), None, s.ring.tolist(), s.state.tolist(), PAGE, ROWS)
        if captured:
            graph.replay()
            torch.cuda.synchronize()
            assert s.err.item() == 0
        else:
            s.by_session(session)
        for t, w in zip((s.table, s.ring, s.held, s.state, s.offsets, s.seqs, s.positions, s.slots), want):
            assert t.tolist() == w
        assert not want[-1]
        offsets = want[4]
        waited += sum(c > 0 and offsets[b + 1] == offsets[b] for b, c in enumerate(counts))
        # the normed heads, and the values as they were
        heads, y = H + HKV, s.x.cpu()
        wanted, err = nr.forward(x[:, :heads * D].contiguous(), s.positions.cpu()[:, None], heads, D,
                                 nr.gammas(heads, HKV, D, s.qg.cpu(), s.kg.cpu()), 1e-6, ([D // 2], D, 1e4, False, False))
        got = y[:, :heads * D].double().reshape(ROWS, heads, D)
        assert bool(((got - wanted).abs() <= ref.half_step(wanted, BF16) + err).all())
        assert ref.same_bits(y[:, heads * D:], x[:, heads * D:])
        # the pages hold them at the planned slots
        for r in range(offsets[-1]):
            kv = y[r, H * D:].view(2, HKV, D)
            known.held[s.seqs[r].item()].append((kv[0], kv[1]))
        at = s.slots.cpu()[:offsets[-1]].long()
        kv = y[:offsets[-1], H * D:].view(-1, 2, HKV, D)
        assert ref.same_bits(s.k.cpu()[at // PAGE, :, at % PAGE], kv[:, 0]) and ref.same_bits(s.v.cpu()[at // PAGE, :, at % PAGE], kv[:, 1])
        assert s.lengths.tolist() == known.lens
        # and every row attends to what its sequence holds
        want, wlse, err, ds = tiles_ref.window(known, y[:, :H * D].contiguous(), H, offsets, WIN, SINKS)
        mine = slice(0, offsets[-1])
        got = s.out.cpu().double().view(ROWS, H, D)
        assert bool(((got - want).abs()[mine] <= (ref.half_step(want, BF16) + err)[mine]).all())
        assert bool(((s.lse.cpu().double() - wlse).abs()[mine] <= ds + 2.0 ** -18 * (1 + wlse[mine].abs())).all())
        assert bool((got[offsets[-1]:] == 7).all()) and bool((s.lse[offsets[-1]:] == 7).all())
    assert waited > 0 and ended > 0 and max(known.lens) > WIN
    del graph


def test_drafts_behind_one_text(session):
    """A text enters pages once, as a sequence of a view of its own, and several drafts grow behind it: each step's
    attention is that of the text and the draft's own rows under one softmax."""
    length, drafts, steps = 45, 3, 12
    g = torch.Generator().manual_seed(3)
    pages = 6 + drafts * 2 + 1
    k = torch.full((pages, HKV, PAGE, D), math.nan, dtype=BF16, device="cuda")
    v = k.clone()
    order = torch.randperm(pages, generator=g).int()
    text, table, lengths = order[None, :6].cuda().contiguous(), order[6:12].view(drafts, 2).cuda(), i32([0] * drafts)
    tlen, text_len = i32([0]), i32([length])
    rows = torch.randn(length, 2 * HKV * D, generator=g).to(BF16)
    known = [[[r.view(2, HKV, D)[i] for i in range(2)] for r in rows] for _ in range(drafts)]
    with ref.Buffers(session) as R:
        bk, bv, x = R(k), R(v), R(rows.cuda())
        one = capi.paged_cache(bk, bv, R(text), R(tlen))
        session.paged_store(one, x, x, v_col=HKV * D, offsets=R(i32([0, length])))
        cache = capi.paged_cache(bk, bv, R(table), R(lengths))
        new = torch.zeros(drafts, W, dtype=BF16, device="cuda")
        out, lse = torch.zeros(drafts, H * D, dtype=BF16, device="cuda"), torch.zeros(drafts, H, device="cuda")
        size = capi.paged_prefix_attention_workspace_bytes(drafts, H, HKV, D, 2 * PAGE, 6 * PAGE)
        bn, bo, bl, ws, pages_id, len_id = R(new), R(out), R(lse), R.workspace(size), R(text.view(-1)), R(text_len)
        for step in range(steps):
            new.copy_(torch.randn(drafts, W, generator=g).to(BF16))
            session.paged_store(cache, bn, bn, k_col=H * D, v_col=(H + HKV) * D)
            session.paged_prefix_attention(cache, pages_id, len_id, bn, bo, H, lse=bl, workspace=ws)
            assert session.device_errors() == 0
            kv = new.cpu()[:, H * D:].view(drafts, 2, HKV, D)
            for b in range(drafts):
                known[b].append([kv[b, 0], kv[b, 1]])
            r = Rows()
            r.held = known
            want, wlse, err, ds = tiles_ref.window(r, new[:, :H * D].contiguous(), H, None, 0, 0)
            got = out.cpu().double().view(drafts, H, D)
            assert bool(((got - want).abs() <= ref.half_step(want, BF16) + err).all())
            assert bool(((lse.cpu().double() - wlse).abs() <= ds + 2.0 ** -18 * (1 + wlse.abs())).all())
    assert tlen.tolist() == [length] and lengths.tolist() == [steps] * drafts
