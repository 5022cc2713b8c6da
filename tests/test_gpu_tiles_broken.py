"""Offsets that cannot be, where rows' keys are cut into parts that a second
kernel adds up: nothing is written, whatever the workspace holds."""
import pytest
import torch

from fercuda_b200 import capi
from tests import paged_ref as ref
from tests.test_gpu_paged_tiles import ERR_BAD, F16, MARK, check_window, i32, queries

pytestmark = pytest.mark.gpu

LENS, HEADS = [20000, 9000, 12345, 7000], 4


def cache():
    """Long sequences over a few pages that they share."""
    c = ref.Cache([64 * 8], 2, 64, 64, F16)
    g = torch.Generator().manual_seed(1)
    c.lens, c.max_pages, c.slots = LENS, 512, 512 * 64
    c.table = torch.randint(0, 8, (len(LENS), 512), generator=g, dtype=torch.int32).cuda()
    held = torch.where(torch.isnan(c.k), 0, c.k), torch.where(torch.isnan(c.v), 0, c.v)
    c.k, c.v = held
    c.lengths = i32(LENS)
    return c


@pytest.mark.parametrize("offsets", [[0, 2, 4, 3, 8], [0, 2, 1, 6, 8], [-1, 2, 4, 6, 8], [0, 2, 4, 6, 9], [0, 9, 4, 6, 8],
                                     [0, 2, 4, 6, 2 ** 31 - 1], [8, 6, 4, 2, 0]])
def test_bad_offsets_leave_results_as_they_were(session, offsets):
    c, rows, D = cache(), 8, 64
    q = queries(rows, HEADS * D, F16)
    out, lse = torch.full((rows, HEADS * D), MARK, dtype=F16, device="cuda"), torch.full((rows, HEADS), MARK, device="cuda")
    size = capi.paged_window_attention_workspace_bytes(rows, len(LENS), HEADS, 2, D, c.slots, 0, 0)
    assert size > rows * HEADS * 4 * D   # there are parts
    with ref.Buffers(session) as B:
        # what an earlier call may have left: a part of every row that counts
        ws = B(torch.ones(size // 4, device="cuda").view(torch.uint8))
        ids, bq, bo, bl = c.ids(B), B(q), B(out), B(lse)
        session.paged_window_attention(ids, bq, bo, HEADS, 0, 0, offsets=B(i32(offsets)), lse=bl, workspace=ws)
        torch.cuda.synchronize()
        assert session.device_errors() == ERR_BAD
        assert bool((out == MARK).all()) and bool((lse == MARK).all())
        # and a call with good ones over the same workspace is as ever, behind it and before it
        good = B(i32([0, 2, 4, 6, 8]))
        session.paged_window_attention(ids, bq, bo, HEADS, 0, 0, offsets=good, lse=bl, workspace=ws)
        torch.cuda.synchronize()
        assert session.device_errors() == 0
        first = out.clone()
        session.paged_window_attention(ids, bq, bo, HEADS, 0, 0, offsets=B(i32(offsets)), lse=bl, workspace=ws)
        torch.cuda.synchronize()
        assert session.device_errors() == ERR_BAD and ref.same_bits(out, first)
    out2, _ = check_window(session, c, q, HEADS, [0, 2, 4, 6, 8], 0, 0)
    assert ref.same_bits(out2, first)
