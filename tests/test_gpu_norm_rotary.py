"""fer_submit_norm_rotary and its gradient against the formulas in 64 bits.

f32 arithmetic: the mean of D squares is off by at most D 2^-24 of itself, the
inverse root by half of that and 2^-22, the products with it and gamma by 2^-23,
turning as in tests/test_gpu_rotary.py by 2^-21 + 2^-22 and, for arguments far
away, 2^-50 times the angle, of twice the head's largest element. A result is then
rounded once. The gradient has the same parts: h by the turn and a product, the
mean of h x by D 2^-23 of the mean of absolute products."""
import pytest
import torch

from fercuda_b200 import capi
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def setup(rows, heads, D, dtype, axes, seed=0, far=50_000, extra=0):
    g = torch.Generator().manual_seed(seed + rows)
    size = torch.exp(torch.randn(heads * D + extra, generator=g))
    x = (torch.randn(rows, heads * D + extra, generator=g) * size).to(dtype)
    dy = torch.randn(rows, heads * D, generator=g).to(dtype)
    pos = torch.randint(0, far, (rows, axes), generator=g, dtype=torch.int32)
    qg, kg = (1 + 0.3 * torch.randn(D, generator=g) for _ in range(2))
    return x, dy, pos, qg, kg


def gammas(heads, k_heads, D, qg, kg):
    one = torch.ones(D, dtype=torch.float64)
    q, k = (one if t is None else t.double() for t in (qg, kg))
    return torch.stack([q] * (heads - k_heads) + [k] * k_heads)


def forward(x, pos, heads, D, gamma, eps, turn):
    x = x.double().view(x.shape[0], heads, D)
    z = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * gamma
    y, far = ref.rotary(z.reshape(x.shape[0], -1), pos, heads, D, *turn, False)
    rel = D * 2.0 ** -25 + 2.0 ** -22 + 2.0 ** -23 + 2.0 ** -22 + 2.0 ** -21 + far[:, None, None] * 2.0 ** -50
    return y, 2 * z.abs().amax(-1, keepdim=True) * rel


def gradient(x, dy, pos, heads, D, gamma, eps, turn):
    rows = x.shape[0]
    x = x.double().view(rows, heads, D)
    g, far = ref.rotary(dy, pos, heads, D, *turn, True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    h = g * gamma
    dx = r * (h - x * r * r * (h * x).mean(-1, keepdim=True))
    rel = D * 2.0 ** -23 + 2.0 ** -20 + far[:, None, None] * 2.0 ** -49
    big = dy.double().view(rows, heads, D).abs().amax(-1, keepdim=True) * 2 * gamma.abs()
    err = rel * r * (big + x.abs() * r * r * (big * x.abs()).mean(-1, keepdim=True))
    unit = x * r
    big = dy.double().view(rows, heads, D).abs().amax(-1, keepdim=True) * 2 * unit.abs()
    # a lane adds the heads of its rows (148 CTAs of 8 warps at least share them out), a CTA its warps, in f32
    terms = -(-rows // (148 * 8)) * heads + 64
    return dx, err, g * unit, (big * rel).sum(0) + terms * 2.0 ** -24 * (g * unit).abs().sum(0)


def call(session, x, out, pos, heads, D, k_heads=0, qg=None, kg=None, **kw):
    with ref.Buffers(session) as B:
        bx = B(x)
        session.norm_rotary(bx, bx if out is x else B(out), B(pos), heads, D, k_heads=k_heads, q_gamma=B(qg), k_gamma=B(kg), **kw)
    assert session.device_errors() == 0


def call_grad(session, x, dy, out, pos, heads, D, dq=None, dk=None, k_heads=0, qg=None, kg=None, **kw):
    with ref.Buffers(session) as B:
        bx, bg = B(x), B(dy)
        bo = bx if out is x else bg if out is dy else B(out)
        session.norm_rotary_grad(bx, bg, bo, B(pos), heads, D, k_heads=k_heads, q_gamma=B(qg), k_gamma=B(kg), q_gamma_grad=B(dq),
                                 k_gamma_grad=B(dk), workspace=B.workspace(capi.norm_rotary_grad_workspace_bytes(x.shape[0], heads, D)),
                                 **kw)
    assert session.device_errors() == 0


# rows, heads, of them keys, head_dim, sections, turned, side by side, frequencies of an axis
SHAPES = [
    (1, 2, 1, 64, [32], 64, False, False),
    (1, 1, 0, 2, [1], 2, True, False),
    (3, 5, 5, 64, [8, 12, 12], 64, False, False),
    (7, 3, 1, 80, [20, 0, 16], 72, False, True),
    (33, 9, 4, 96, [31], 62, False, False),          # an odd half: one element at a time
    (33, 9, 4, 98, [31], 62, True, False),
    (65, 40, 8, 128, [64], 128, False, False),
    (129, 6, 2, 256, [1, 2, 3, 122], 256, True, True),
    (40, 7, 3, 250, [62], 124, True, False),
    (40, 7, 3, 254, [63], 126, False, False),
    (11, 130, 65, 32, [16], 32, False, False),
    (2500, 5, 2, 64, [32], 64, False, False),         # rows enough for copies
    (2500, 3, 1, 128, [20], 40, False, False),        # and a tail
    (2401, 9, 4, 128, [24, 40], 128, True, False),
    (2600, 2, 1, 256, [60], 120, True, False),
    (2500, 40, 8, 128, [64], 128, False, False),      # parts of a row
    (2400, 47, 7, 80, [40], 80, False, False),        # the last part has fewer heads
    (3001, 33, 16, 48, [8, 8], 32, False, False),
    (2400, 3, 1, 66, [33], 66, False, False),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,heads,k_heads,D,sections,rot,inter,freqs", SHAPES)
def test_matches_definition(session, dtype, rows, heads, k_heads, D, sections, rot, inter, freqs):
    x, dy, pos, qg, kg = setup(rows, heads, D, dtype, len(sections))
    turn = (sections, rot, 5e5, inter, freqs)
    kw = dict(k_heads=k_heads, qg=qg.cuda(), kg=kg.cuda(), sections=sections, rotary_dim=rot, base=5e5, interleaved=inter,
              axis_freqs=freqs, eps=1e-5)
    gamma = gammas(heads, k_heads, D, qg, kg)
    out = torch.full_like(x, 7.0).cuda()
    call(session, x.cuda(), out, pos.cuda(), heads, D, **kw)
    want, err = forward(x, pos, heads, D, gamma, 1e-5, turn)
    assert bool(((out.cpu().double().view_as(want) - want).abs() <= ref.half_step(want, dtype) + err).all())

    dx = torch.full_like(x, 7.0).cuda()
    dq, dk = torch.full((D,), 7.0).cuda(), torch.full((D,), 7.0).cuda()
    call_grad(session, x.cuda(), dy.cuda(), dx, pos.cuda(), heads, D, dq, dk, **kw)
    want, err, each, gerr = gradient(x, dy, pos, heads, D, gamma, 1e-5, turn)
    assert bool(((dx.cpu().double().view_as(want) - want).abs() <= ref.half_step(want, dtype) + err).all())
    each = each.sum(0)
    for got, part in ((dq, slice(0, heads - k_heads)), (dk, slice(heads - k_heads, heads))):
        w = each[part].sum(0)
        assert bool(((got.cpu().double() - w).abs() <= gerr[part].sum(0) + ref.half_step(w, F32)).all())


@pytest.mark.parametrize("rows", [5, 2500])
@pytest.mark.parametrize("which", ["q", "k", "none"])
def test_gammas_that_are_left_out(session, rows, which):
    x, dy, pos, qg, kg = setup(rows, 4, 64, BF16, 1)
    qg, kg = (qg if which == "q" else None), (kg if which == "k" else None)
    turn, dev = ([32], 64, 1e4, False, False), lambda t: None if t is None else t.cuda()
    out, dx = torch.zeros_like(x).cuda(), torch.zeros_like(x).cuda()
    call(session, x.cuda(), out, pos.cuda(), 4, 64, 1, dev(qg), dev(kg))
    want, err = forward(x, pos, 4, 64, gammas(4, 1, 64, qg, kg), 1e-6, turn)
    assert bool(((out.cpu().double().view_as(want) - want).abs() <= ref.half_step(want, BF16) + err).all())
    only = torch.zeros(64, device="cuda")
    call_grad(session, x.cuda(), dy.cuda(), dx, pos.cuda(), 4, 64, None, only, 1, dev(qg), dev(kg))
    want, err, each, gerr = gradient(x, dy, pos, 4, 64, gammas(4, 1, 64, qg, kg), 1e-6, turn)
    assert bool(((dx.cpu().double().view_as(want) - want).abs() <= ref.half_step(want, BF16) + err).all())
    w = each.sum(0)[3]
    assert bool(((only.cpu().double() - w).abs() <= gerr[3] + ref.half_step(w, F32)).all())


@pytest.mark.parametrize("rows", [3, 2500])
def test_rows_of_zeros(session, rows):
    """With eps they give zeros and the gradient's r = eps^-1/2; without, 0 / 0 is NaN in that head alone."""
    x, dy, pos, qg, kg = setup(rows, 3, 64, F32, 1)
    x[1, 64:128] = 0
    out, dx = torch.zeros_like(x).cuda(), torch.zeros_like(x).cuda()
    call(session, x.cuda(), out, pos.cuda(), 3, 64, eps=1e-6)
    assert bool((out[1, 64:128] == 0).all()) and bool(out.isfinite().all())
    call_grad(session, x.cuda(), dy.cuda(), dx, pos.cuda(), 3, 64, eps=1e-6)
    want, err, _, _ = gradient(x, dy, pos, 3, 64, gammas(3, 0, 64, None, None), 1e-6, ([32], 64, 1e4, False, False))
    assert bool(((dx.cpu().double().view_as(want) - want).abs() <= ref.half_step(want, F32) + err).all())
    call(session, x.cuda(), out, pos.cuda(), 3, 64, eps=0.0)
    assert bool(out[1, 64:128].isnan().all())
    out[1, 64:128] = 0
    assert bool(out.isfinite().all())


@pytest.mark.parametrize("dtype,x_col,out_col,g_col,extra", [
    (BF16, 0, 0, 0, 16), (BF16, 8, 16, 8, 24), (F16, 1, 3, 5, 6), (F32, 4, 8, 12, 16), (F32, 2, 1, 3, 5), (BF16, 2, 6, 4, 8)])
@pytest.mark.parametrize("rows", [9, 2400])
@pytest.mark.parametrize("inter", [False, True])
def test_columns_of_wider_rows(session, dtype, x_col, out_col, g_col, extra, rows, inter):
    heads, D, W = 3, 64, 3 * 64
    x, _, pos, qg, kg = setup(rows, heads, D, dtype, 1, extra=extra + 16)
    dy = setup(rows, heads, D, dtype, 1, seed=9, extra=extra + 16)[0]
    kw = dict(k_heads=1, qg=qg.cuda(), kg=kg.cuda(), interleaved=inter)
    gamma, turn = gammas(heads, 1, D, qg, kg), ([32], 64, 1e4, inter, False)
    px, pg = x[:, x_col: x_col + W].contiguous(), dy[:, g_col: g_col + W].contiguous()
    for grad in (False, True):
        out = torch.full((rows, W + extra + 16), 9.0, dtype=dtype).cuda()
        if grad:
            call_grad(session, x.cuda(), dy.cuda(), out, pos.cuda(), heads, D, x_col=x_col, out_col=out_col, grad_col=g_col, **kw)
            want, err, _, _ = gradient(px, pg, pos, heads, D, gamma, 1e-6, turn)
        else:
            call(session, x.cuda(), out, pos.cuda(), heads, D, x_col=x_col, out_col=out_col, **kw)
            want, err = forward(px, pos, heads, D, gamma, 1e-6, turn)
        got = out.cpu()
        part = got[:, out_col: out_col + W].double().reshape(want.shape)
        assert bool(((part - want).abs() <= ref.half_step(want, dtype) + err).all())
        assert bool((got[:, :out_col] == 9).all()) and bool((got[:, out_col + W:] == 9).all())


@pytest.mark.parametrize("rows,heads,D,rot", [(50, 6, 64, 64), (2500, 6, 64, 40), (2500, 40, 128, 128), (300, 5, 62, 62)])
def test_in_place_gives_the_same_bits(session, rows, heads, D, rot):
    x, dy, pos, qg, kg = setup(rows, heads, D, BF16, 1)
    x, dy, pos, kw = x.cuda(), dy.cuda(), pos.cuda(), dict(k_heads=2, qg=qg.cuda(), kg=kg.cuda(), rotary_dim=rot)
    out = torch.empty_like(x)
    call(session, x, out, pos, heads, D, **kw)
    here = x.clone()
    call(session, here, here, pos, heads, D, **kw)
    assert ref.same_bits(here, out)
    sums = [torch.zeros(D, device="cuda") for _ in range(6)]
    call_grad(session, x, dy, out, pos, heads, D, sums[0], sums[1], **kw)
    here = x.clone()
    call_grad(session, here, dy, here, pos, heads, D, sums[2], sums[3], **kw)
    assert ref.same_bits(here, out)
    here = dy.clone()
    call_grad(session, x, here, here, pos, heads, D, sums[4], sums[5], **kw)
    assert ref.same_bits(here, out)
    assert all(ref.same_bits(sums[i], sums[i + 2]) for i in range(4))


@pytest.mark.parametrize("rows", [6, 2400])
def test_gradient_against_differences(session, rows):
    """Central differences of the 64-bit forward along random directions: off by step^2 of its third derivative."""
    heads, D, secs = 3, 64, [8, 8, 16]
    x, dy, pos, qg, kg = setup(rows, heads, D, F32, 3, far=500)
    x = x / x.abs().amax() + 0.1 * torch.randn(x.shape, generator=torch.Generator().manual_seed(8))
    dx, dq, dk = torch.empty_like(x).cuda(), torch.empty(D).cuda(), torch.empty(D).cuda()
    call_grad(session, x.cuda(), dy.cuda(), dx, pos.cuda(), heads, D, dq, dk, k_heads=1, qg=qg.cuda(), kg=kg.cuda(), sections=secs,
              eps=1e-2)
    turn = (secs, D, 1e4, False, False)

    def loss(x, qg, kg):
        y, _ = forward(x, pos, heads, D, gammas(heads, 1, D, qg, kg), 1e-2, turn)
        return float((y.reshape(rows, -1) * dy.double()).sum())

    g = torch.Generator().manual_seed(77)
    step = 1e-4
    x, qg, kg = x.double(), qg.double(), kg.double()
    for i, (got, at) in enumerate(((dx, 0), (dq, 1), (dk, 2))):
        d = torch.randn([x, qg, kg][at].shape, generator=g, dtype=torch.float64)
        up, dn = [x, qg, kg], [x, qg, kg]
        up[at], dn[at] = up[at] + step * d, dn[at] - step * d
        slope = (loss(*up) - loss(*dn)) / (2 * step)
        terms = got.cpu().double() * d
        # f32 results (each within 2^-15 of the largest), and differences in 64 bits: step^2 and rounding / step
        size = float(terms.abs().sum())
        assert abs(float(terms.sum()) - slope) <= size * (2.0 ** -15 + 1e-6) + 1e-6 * rows ** 0.5


def test_the_same_bits_every_time(session):
    x, dy, pos, qg, kg = (t.cuda() for t in setup(5000, 12, 128, BF16, 1))
    first = None
    for _ in range(4):
        dx, dq, dk = torch.empty_like(x), torch.empty(128, device="cuda"), torch.empty(128, device="cuda")
        call_grad(session, x, dy, dx, pos, 12, 128, dq, dk, k_heads=4, qg=qg, kg=kg)
        first = first or (dx, dq, dk)
        assert all(ref.same_bits(a, b) for a, b in zip(first, (dx, dq, dk)))


def test_rows_behind_two_to_the_31_elements(session):
    rows, width = 2400, 1 << 20
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    few, dy, pos, qg, kg = setup(rows, 3, 64, BF16, 1)
    x = torch.zeros(rows, width, dtype=BF16, device="cuda")
    x[:, -192:] = few.cuda()
    out = torch.empty(rows, 192, dtype=BF16, device="cuda")
    want = torch.empty_like(out)
    kw = dict(k_heads=1, qg=qg.cuda(), kg=kg.cuda())
    call(session, few.cuda(), want, pos.cuda(), 3, 64, **kw)
    call(session, x, out, pos.cuda(), 3, 64, x_col=width - 192, **kw)
    assert ref.same_bits(out, want)
    call_grad(session, few.cuda(), dy.cuda(), want, pos.cuda(), 3, 64, **kw)
    call_grad(session, x, dy.cuda(), out, pos.cuda(), 3, 64, x_col=width - 192, **kw)
    assert ref.same_bits(out, want)
    del x
    torch.cuda.empty_cache()


def test_no_rows(session):
    one = torch.zeros(1, 128, dtype=BF16, device="cuda")
    args = capi.fer_norm_rotary_args_t
    a = args()
    a.rotary = capi.fer_rotary_args_t(one.data_ptr(), one.data_ptr(), one.data_ptr(), 128, 128, 0, 2, 64, 64, 1, (32,), 1e4, 0,
                                      capi.FER_DTYPE_BF16)
    a.eps = 1e-6
    dq, ws = torch.full((64,), 7.0, device="cuda"), torch.zeros(64, device="cuda")
    d = capi.fer_norm_rotary_grad_t(one.data_ptr(), 128, dq.data_ptr(), None, ws.data_ptr(), 256)
    import ctypes as C
    s = torch.cuda.current_stream().cuda_stream
    assert capi.kernels().fer_norm_rotary(C.byref(a), None, s) == 0
    assert capi.kernels().fer_norm_rotary_grad(C.byref(a), C.byref(d), None, s) == 0
    torch.cuda.synchronize()
    assert bool((dq == 0).all())


def test_captured_on_two_streams(session):
    """A backward pass captured with a workspace of its own and replayed beside an eager one."""
    import ctypes as C
    rows, heads, D = 2500, 6, 128
    x, dy, pos, qg, kg = (t.cuda() for t in setup(rows, heads, D, F16, 1))
    a = capi.fer_norm_rotary_args_t()
    a.k_heads, a.q_gamma, a.k_gamma, a.eps = 2, qg.data_ptr(), kg.data_ptr(), 1e-6
    made = []

    def go(stream):
        dx, dq, dk = torch.zeros_like(x), torch.zeros(D, device="cuda"), torch.zeros(D, device="cuda")
        ws = torch.full((capi.norm_rotary_grad_workspace_bytes(rows, heads, D),), 255, dtype=torch.uint8, device="cuda")
        a.rotary = capi.fer_rotary_args_t(x.data_ptr(), dx.data_ptr(), pos.data_ptr(), heads * D, heads * D, rows, heads, D, D, 1,
                                          (D // 2,), 1e4, 0, capi.FER_DTYPE_F16)
        d = capi.fer_norm_rotary_grad_t(dy.data_ptr(), heads * D, dq.data_ptr(), dk.data_ptr(), ws.data_ptr(), ws.numel())
        made.append((dx, dq, dk, ws))
        assert capi.kernels().fer_norm_rotary_grad(C.byref(a), C.byref(d), None, stream) == 0

    go(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        go(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        graph.replay()
        with torch.cuda.stream(side):
            go(side.cuda_stream)
    torch.cuda.synchronize()
    for other in made[1:]:
        assert all(ref.same_bits(p, q) for p, q in zip(made[0][:3], other[:3]))
    del graph


@pytest.mark.parametrize("change,word", [
    (dict(k_heads=5), "key heads"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(q_gamma="short"), "gammas"), (dict(q_gamma="x"), "gammas"), (dict(k_gamma="over"), "overlap"), (dict(head_dim=512), "head_dim"),
    (dict(out="shift"), "overlap"), (dict(x_col=1), "columns"), (dict(sections=(3,)), "sections"), (dict(base=0.0), "base"),
    (dict(positions="x"), "positions"), (dict(rotary_dim=66), "rotary_dim")])
def test_refusals(session, change, word):
    x, _, pos, qg, kg = (t.cuda() for t in setup(4, 4, 64, F32, 1))
    other, wide = torch.zeros_like(x), torch.zeros(4, 4 * 64 + 64, device="cuda")
    with ref.Buffers(session) as B:
        bufs = dict(x=B(x), out=B(other), positions=B(pos), q_gamma=B(qg), k_gamma=B(kg), short=B(qg[:60].contiguous()),
                    wide=B(wide), over=session.import_ptr(capi.FER_DTYPE_F32, [64], other.data_ptr() + 256))
        B.ids.append(bufs["over"])
        kw = dict(sections=change.get("sections", (0,)), eps=change.get("eps", 1e-6), base=change.get("base", 1e4),
                  k_heads=change.get("k_heads", 1), x_col=change.get("x_col", 0), rotary_dim=change.get("rotary_dim", 0))
        pick = lambda n: bufs[change.get(n, n)]  # noqa: E731
        with pytest.raises(capi.FerError) as e:
            if change.get("out") == "shift":
                session.norm_rotary(bufs["wide"], bufs["wide"], bufs["positions"], 4, 64, out_col=32, **kw)
            else:
                session.norm_rotary(pick("x"), pick("out"), pick("positions"), 4, change.get("head_dim", 64), q_gamma=pick("q_gamma"),
                                    k_gamma=pick("k_gamma"), **kw)
    assert e.value.code == capi.FER_STATUS_INVALID_ARGUMENT and word in e.value.msg, e.value.msg


@pytest.mark.parametrize("change,word", [
    (dict(grad="pos"), "grad"), (dict(grad="few"), "grad"), (dict(grad_col=1), "columns"), (dict(dq="short"), "gradients"),
    (dict(dq="dk"), "overlap"), (dict(dq="q_gamma"), "overlap"), (dict(ws="small"), "workspace"), (dict(ws="dk"), "workspace"),
    (dict(dk="in_out"), "overlap"), (dict(eps=-1.0), "eps")])
def test_gradient_refusals(session, change, word):
    x, dy, pos, qg, kg = (t.cuda() for t in setup(4, 4, 64, F32, 1))
    other = torch.zeros_like(x)
    with ref.Buffers(session) as B:
        bufs = dict(x=B(x), grad=B(dy), out=B(other), pos=B(pos), q_gamma=B(qg), dq=B(torch.zeros(64, device="cuda")),
                    dk=B(torch.zeros(64, device="cuda")), ws=B.workspace(1 << 20), small=B.workspace(64),
                    few=B(torch.zeros(3, 256, device="cuda")), short=B(torch.zeros(60, device="cuda")),
                    in_out=session.import_ptr(capi.FER_DTYPE_F32, [64], other.data_ptr() + 512))
        B.ids.append(bufs["in_out"])
        pick = lambda n: bufs[change.get(n, n)]  # noqa: E731
        with pytest.raises(capi.FerError) as e:
            session.norm_rotary_grad(bufs["x"], pick("grad"), bufs["out"], bufs["pos"], 4, 64, workspace=pick("ws"), k_heads=1,
                                     q_gamma=bufs["q_gamma"], q_gamma_grad=pick("dq"), k_gamma_grad=pick("dk"),
                                     grad_col=change.get("grad_col", 0), eps=change.get("eps", 1e-6))
    assert e.value.code == capi.FER_STATUS_INVALID_ARGUMENT and word in e.value.msg, e.value.msg
