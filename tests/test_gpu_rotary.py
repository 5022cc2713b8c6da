"""fer_submit_rotary against the definition in 64 bits.

Tolerance of a result y = a cos - b sin: half a step of its type, plus for the
f32 arithmetic (|a| + |b|) times (2^-22 for the two products and their sum, 2^-21
for cosine and sine with an argument rounded to f32, and 2^-50 times the angle
for the 64-bit frequency and product, in the oracle as well)."""
import numpy as np
import pytest
import torch

from fercuda_b200 import capi
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def bound(x, y, far, dtype, heads, head_dim):
    mag = x.double().abs().view(x.shape[0], heads, head_dim).amax(-1, keepdim=True) * 2
    return ref.half_step(y, dtype) + mag * (2.0 ** -22 + 2.0 ** -21 + far[:, None, None] * 2.0 ** -50)


def call(session, x, out, pos, heads, head_dim, **kw):
    with ref.Buffers(session) as B:
        bx = B(x)
        session.rotary(bx, bx if out is x else B(out), B(pos), heads, head_dim, **kw)
    assert session.device_errors() == 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,heads,head_dim,sections,rot,inter,freqs,inv", [
    (1, 1, 64, [32], 64, False, False, False),
    (1, 5, 2, [1], 2, True, False, False),
    (3, 2, 64, [8, 12, 12], 64, False, False, True),
    (7, 3, 128, [16, 24, 24], 128, True, False, False),
    (65, 4, 128, [32, 32], 128, False, True, False),
    (33, 2, 80, [20, 0, 16], 72, False, False, False),     # an axis without pairs, a tail that is copied
    (33, 2, 80, [1, 2, 3, 31], 74, True, True, True),
    (129, 7, 96, [31], 62, False, False, False),           # odd half: one element at a time
    (257, 1, 256, [128], 256, False, False, False),
    (1000, 40, 64, [16, 16], 64, False, True, False),
    (5, 130, 1024, [512], 1024, False, False, False)])
def test_matches_definition(session, dtype, rows, heads, head_dim, sections, rot, inter, freqs, inv):
    g = torch.Generator().manual_seed(rows * 31 + heads)
    x = (torch.randn(rows, heads * head_dim, generator=g) * 3).to(dtype)
    pos = torch.randint(0, 100_000, (rows, len(sections)), generator=g, dtype=torch.int32)
    out = torch.full_like(x, 7.0).cuda()
    call(session, x.cuda(), out, pos.cuda(), heads, head_dim, sections=sections, rotary_dim=rot, base=5e5,
         interleaved=inter, axis_freqs=freqs, inverse=inv)
    want, far = ref.rotary(x, pos, heads, head_dim, sections, rot, 5e5, inter, freqs, inv)
    got = out.cpu().double().view_as(want)
    assert bool(((got - want).abs() <= bound(x, want, far, dtype, heads, head_dim)).all())
    if rot < head_dim:
        assert torch.equal(got[..., rot:], x.double().view_as(want)[..., rot:])


@pytest.mark.parametrize("dtype,rows,heads,head_dim,rot,col", [
    (BF16, 9, 3, 72, 64, 0), (BF16, 9, 3, 72, 64, 1), (F32, 700, 5, 68, 64, 0), (F16, 40, 32, 128, 32, 8),
    (BF16, 3, 9000, 34, 32, 0),            # one piece a head
    (F16, 2, 5000, 1024, 2, 0), (F16, 2, 5000, 1024, 2, 1)])
def test_copied_tails(session, dtype, rows, heads, head_dim, rot, col):
    """What lies behind the turned part arrives as it is, and nothing is written beside the heads."""
    g = torch.Generator().manual_seed(heads)
    x = torch.randn(rows, heads * head_dim + 16, generator=g).to(dtype).cuda()
    pos = torch.randint(0, 5000, (rows,), generator=g, dtype=torch.int32)
    out = torch.full_like(x, 7.0)
    call(session, x, out, pos.cuda(), heads, head_dim, rotary_dim=rot, x_col=col, out_col=col)
    part = slice(col, col + heads * head_dim)
    got, src = out[:, part].reshape(rows, heads, head_dim), x[:, part].reshape(rows, heads, head_dim)
    assert ref.same_bits(got[..., rot:], src[..., rot:])
    rest = out.clone()
    rest[:, part] = 7.0
    assert bool((rest == 7.0).all())
    want, far = ref.rotary(src.cpu().view(rows, -1), pos[:, None], heads, head_dim, [rot // 2], rot, 1e4, False, False, False)
    assert bool(((got.cpu().double() - want).abs() <= bound(src.cpu().view(rows, -1), want, far, dtype, heads, head_dim)).all())


def test_far_and_negative_positions(session):
    pos = torch.tensor([0, 1, -1, 12345, -99999, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    x = torch.randn(8, 64, generator=torch.Generator().manual_seed(1))
    out = torch.empty_like(x).cuda()
    call(session, x.cuda(), out, pos.cuda(), 1, 64)
    want, far = ref.rotary(x, pos[:, None], 1, 64, [32], 64, 1e4, False, False, False)
    assert bool(((out.cpu().double().view_as(want) - want).abs() <= bound(x, want, far, F32, 1, 64)).all())
    assert torch.equal(out[0].cpu(), x[0])                 # position 0 turns nothing


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("x_col,out_col,extra", [(0, 0, 0), (1, 3, 5), (8, 4, 16), (2, 2, 2)])
def test_columns_of_wider_rows(session, inter, x_col, out_col, extra):
    rows, heads, D = 19, 3, 64
    g = torch.Generator().manual_seed(3)
    x = torch.randn(rows, x_col + heads * D + extra, generator=g).to(BF16)
    out = torch.full((rows, out_col + heads * D + 3), 9.0, dtype=BF16)
    pos = torch.randint(0, 999, (rows,), generator=g, dtype=torch.int32)
    dev = out.cuda()
    call(session, x.cuda(), dev, pos.cuda(), heads, D, x_col=x_col, out_col=out_col, interleaved=inter)
    part = x[:, x_col:x_col + heads * D].contiguous()
    want, far = ref.rotary(part, pos[:, None], heads, D, [32], D, 1e4, inter, False, False)
    got = dev.cpu()
    assert bool(((got[:, out_col:out_col + heads * D].double().reshape(want.shape) - want).abs()
                 <= bound(part, want, far, BF16, heads, D)).all())
    assert bool((got[:, :out_col] == 9).all()) and bool((got[:, out_col + heads * D:] == 9).all())


@pytest.mark.parametrize("rot", [64, 40])
def test_in_place_gives_the_same_bits(session, rot):
    rows, heads, D = 300, 6, 64
    g = torch.Generator().manual_seed(4)
    x = torch.randn(rows, heads * D + 128, generator=g).to(F16).cuda()
    pos = torch.randint(0, 4096, (rows,), generator=g, dtype=torch.int32).cuda()
    out = x.clone()
    call(session, x.clone(), out, pos, heads, D, x_col=64, out_col=64, rotary_dim=rot)
    here = x.clone()
    call(session, here, here, pos, heads, D, x_col=64, out_col=64, rotary_dim=rot)
    assert ref.same_bits(here, out)


def test_inverse_is_the_gradient(session):
    """With f(x) = sum(g . rotate(x)) the gradient is the inverse of g; against autograd of the formula, and
    against differences along random directions (the map is linear, so they differ by rounding alone)."""
    rows, heads, D, secs = 11, 2, 64, [8, 8, 16]
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(rows, heads * D, generator=gen, dtype=torch.float64, requires_grad=True)
    gr = torch.randn(rows, heads * D, generator=gen)
    pos = torch.randint(0, 500, (rows, 3), generator=gen, dtype=torch.int32)
    y, far = ref.rotary(x.clone(), pos, heads, D, secs, D, 1e4, False, False, False)
    (y.view(rows, -1) * gr.double()).sum().backward()
    out = torch.empty_like(gr).cuda()
    call(session, gr.cuda(), out, pos.cuda(), heads, D, sections=secs, inverse=True)
    err = (out.cpu().double() - x.grad).abs().view(rows, heads, D)
    assert bool((err <= bound(gr, x.grad.view(rows, heads, D), far, F32, heads, D)).all())
    for k in range(3):
        step = torch.randn(rows, heads * D, generator=gen)
        fwd = torch.empty_like(step).cuda()
        call(session, step.cuda(), fwd, pos.cuda(), heads, D, sections=secs)
        a = float((fwd.cpu().double() * gr.double()).sum())
        b = float((out.cpu().double() * step.double()).sum())
        # both sums have rows * heads * D terms, each off by less than 2^-20 of a term of their product's size
        assert abs(a - b) <= 2.0 ** -20 * float((step.abs().double() * 2 * gr.abs().double().amax()).sum())


def test_infinities_stay_in_their_pair(session):
    x = torch.ones(1, 64)
    x[0, 3], x[0, 40] = float("inf"), float("nan")
    out = torch.empty_like(x).cuda()
    call(session, x.cuda(), out, torch.tensor([5], dtype=torch.int32).cuda(), 1, 64)
    got = out.cpu()[0]
    for i in range(64):
        assert bool(torch.isfinite(got[i])) == (i % 32 not in (3, 8)), i


def test_large_offsets(session):
    """Rows behind 2^31 elements."""
    rows, width = 5, 1 << 29
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GB")
    x = torch.zeros(rows, width, dtype=BF16, device="cuda")
    x[4, -64:] = torch.arange(64, dtype=BF16, device="cuda")
    pos = torch.full((rows,), 3, dtype=torch.int32, device="cuda")
    out = torch.empty(rows, 64, dtype=BF16, device="cuda")
    call(session, x, out, pos, 1, 64, x_col=width - 64)
    want, far = ref.rotary(x[4:, -64:].cpu(), pos[4:, None].cpu(), 1, 64, [32], 64, 1e4, False, False, False)
    assert bool(((out[4:].cpu().double().view_as(want) - want).abs()
                 <= bound(x[4:, -64:].cpu(), want, far, BF16, 1, 64)).all())


@pytest.mark.parametrize("change", [
    dict(heads=3), dict(head_dim=62), dict(head_dim=1026), dict(heads=0), dict(sections=(31,)),
    dict(sections=(16, 16)), dict(rotary_dim=33), dict(rotary_dim=66), dict(base=0.0), dict(base=float("nan")),
    dict(x_col=1), dict(out_col=1), dict(bad="dtype"), dict(bad="rows"), dict(bad="positions"), dict(bad="rank"),
    dict(bad="shifted"), dict(bad="over positions")])
def test_refusals(session, change):
    x = torch.zeros(4, 128, dtype=BF16, device="cuda")
    out, pos = torch.zeros_like(x), torch.zeros(4, dtype=torch.int32, device="cuda")
    kw = dict(heads=2, head_dim=64, sections=(32,))
    bad = change.get("bad")
    kw.update({k: v for k, v in change.items() if k != "bad"})
    if bad == "dtype":
        out = out.to(F16)
    elif bad == "rows":
        out = out[:3].contiguous()
    elif bad == "positions":
        pos = pos.float()
    elif bad == "rank":
        x = x.view(2, 2, 128)
    elif bad == "over positions":
        out = torch.zeros(4, 128, dtype=BF16, device="cuda")
        pos = out.view(torch.int32).view(-1)[:4]
    with ref.Buffers(session) as B:
        ids = [B(x), B(out), B(pos)]
        if bad == "shifted":       # the same memory, one row further
            ids[0] = B(torch.zeros(5, 128, dtype=BF16, device="cuda"))
            whole = B.keep[-1]
            ids[0], ids[1] = B(whole[:4]), B(whole[1:])
        with pytest.raises(capi.FerError) as e:
            session.rotary(*ids, kw.pop("heads"), kw.pop("head_dim"), **kw)
        assert e.value.code == capi.FER_STATUS_INVALID_ARGUMENT
    if bad:
        return
    with pytest.raises(capi.FerError) as e:
        session.rotary(10 ** 9, 10 ** 9, 10 ** 9, 2, 64)
    assert e.value.code == capi.FER_STATUS_NOT_FOUND


def test_many_rows_deterministic(session):
    rows, heads, D = 20011, 4, 64
    x = torch.randn(rows, heads * D, generator=torch.Generator().manual_seed(8)).to(BF16).cuda()
    pos = (torch.arange(rows, dtype=torch.int32) * 7).cuda()
    outs = [torch.empty_like(x) for _ in range(2)]
    for o in outs:
        call(session, x, o, pos, heads, D)
    assert ref.same_bits(*outs)
    pick = torch.from_numpy(np.random.RandomState(1).choice(rows, 200, replace=False))
    want, far = ref.rotary(x.cpu()[pick], pos.cpu()[pick, None], heads, D, [32], D, 1e4, False, False, False)
    assert bool(((outs[0].cpu()[pick].double().view_as(want) - want).abs()
                 <= bound(x.cpu()[pick], want, far, BF16, heads, D)).all())
