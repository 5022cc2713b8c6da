"""Paged-cache operators where a table is full to its last slot and where a
rounding inside a kernel would show, against the 64-bit restatements of
tests/paged_ref.py."""
import pytest
import torch

from tests import paged_ref as ref
from tests import paged_sharp as sharp
from tests.test_gpu_paged import attend, check_evict, run_evict, weights_for

pytestmark = pytest.mark.gpu

ERR_BAD = 4


@pytest.mark.parametrize("batch,slots,cut", [
    # a CTA of 256 threads a head, runs of 12, 20, 24 and 28 slots a thread
    (160, 2176, 30), (160, 4864, 64), (160, 5248, 64), (160, 6400, 64), (160, 4608, 2000),
    # of 1024 threads
    (75, 8320, 64), (75, 20224, 64), (75, 24320, 10000), (75, 28288, 64),
    # clusters of eight, and of four
    (1, 8 * 8320, 100), (1, 8 * 20224, 100), (16, 4 * 8320, 20000)])
def test_evict_from_a_full_table(session, batch, slots, cut):
    """The longest sequences hold every slot of the table's width."""
    lens = [slots] * min(batch, 2) + [40 + b for b in range(batch - 2)]
    lens[-1] = slots
    c = ref.Cache(lens, 1, 64, 64, torch.bfloat16)
    assert c.slots == slots
    w = weights_for("ties" if cut < 100 else "spread", batch, 1, slots, seed=slots).cuda()
    p = torch.arange(slots, dtype=torch.int32, device="cuda").repeat(batch, 1, 1)
    w0, p0 = w.clone(), p.clone()
    before = (c.k.cpu().clone(), c.v.cpu().clone(), w0, p0)
    run_evict(session, c, slots - cut, 50, w, p, c.lengths.clone())
    check_evict(c, slots - cut, 50, w0, p0, torch.tensor(lens, dtype=torch.int32), before, (c.k, c.v, w, p, c.lengths))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,H,group,page", [(64, 2, 1, 8), (64, 1, 9, 16), (128, 2, 4, 64), (128, 1, 16, 8),
                                            (256, 1, 3, 32), (256, 2, 20, 16)])
def test_attention_keeps_probabilities_in_two_parts(session, dtype, D, H, group, page):
    """Scores are exact and values alike in size, so a P rounded once, or a lost
    low part, would go past the bound (tests/test_paged_sharp_bound.py)."""
    c = ref.Cache([1, 2, 3, 5, 8, 13, 16, 33, 64], H, D, page, dtype, seed=D + group)
    q = sharp.fill(c, group, D + group).cuda()
    out, _ = attend(session, c, q, H * group, scale=1.0)
    out = out.cpu().double().view(len(c.lens), H, group, D)
    for b, (p, v) in enumerate(sharp.answers(c, group)):
        assert float((out[b] - p @ v).abs().max()) <= sharp.bound(c, b), (b, c.lens[b])


@pytest.mark.parametrize("bad,becomes", [(-3, 0), (10 ** 6, 64)])
@pytest.mark.parametrize("in_place", [False, True])
def test_store_reports_a_bad_length_without_rows(session, bad, becomes, in_place):
    """A sequence that gets no row has its length clamped; that is reported as any other."""
    c = ref.Cache([20, 30, 64], 2, 64, 16, torch.bfloat16)
    c.lengths[1] = bad
    k, v = c.k.clone(), c.v.clone()
    rows = torch.randn(4, 2 * c.H * c.D, device="cuda").to(c.dtype)
    offsets = torch.tensor([0, 4, 4, 4], dtype=torch.int32, device="cuda")
    new = c.lengths if in_place else torch.full_like(c.lengths, -1)
    with ref.Buffers(session) as B:
        ids, r = c.ids(B), B(rows)
        session.paged_store(ids, r, r, v_col=c.H * c.D, offsets=B(offsets), new_lengths=0 if in_place else B(new))
    assert session.device_errors() == ERR_BAD
    assert new.tolist() == [24, becomes, 64]
    for pool, old, col in ((c.k, k, 0), (c.v, v, c.H * c.D)):
        old[c.table[0, 1].item(), :, 4:8] = rows[:, col: col + c.H * c.D].view(4, c.H, c.D).transpose(0, 1)
        assert ref.same_bits(pool, old)
