"""Attention tiles of few rows keep what rounding P leaves, as documented, and so
do single tokens behind a window and a short batch behind a prefix."""
import pytest
import torch

from fercuda_b200 import capi
from tests import paged_ref as ref
from tests import paged_sharp, tiles_sharp
from tests.test_gpu_paged_tiles import i32

LENS = [1, 2, 3, 5, 8, 13, 16, 33, 64, 130, 200]
# head_dim, key heads, group, page, new rows of each sequence: units of up to 32 rows, and of up to 128 (64 at head_dim 256)
SHAPES = [(64, 2, 1, 8, 2), (64, 1, 3, 16, 7), (128, 2, 4, 64, 8), (128, 1, 16, 8, 2), (256, 1, 3, 32, 10), (256, 2, 20, 16, 1),
          (64, 1, 1, 16, 33), (64, 2, 3, 16, 30), (128, 2, 4, 16, 32), (128, 1, 7, 8, 9), (256, 1, 2, 16, 32), (256, 2, 4, 64, 11)]


def rows_of(lens, new):
    """(row, sequence, slots that it sees): each sequence's last `new` slots, rows without a slot among them."""
    return [(b * new + i, b, n - new + i + 1) for b, n in enumerate(lens) for i in range(new)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,H,group,page,new", SHAPES)
def test_few_rows_keep_probabilities_in_two_parts(session, dtype, D, H, group, page, new):
    c = ref.Cache(LENS, H, D, page, dtype, seed=D + group)
    tiles_sharp.fill(c, group, D + group)
    rows = len(LENS) * new
    q = tiles_sharp.queries(c, group, rows).cuda()
    out = torch.full_like(q, 7.0)
    offsets = i32([b * new for b in range(len(LENS) + 1)])
    with ref.Buffers(session) as B:
        size = capi.paged_window_attention_workspace_bytes(rows, len(LENS), H * group, H, D, c.slots, 0, 0)
        session.paged_window_attention(c.ids(B), B(q), B(out), H * group, 0, 0, offsets=B(offsets), workspace=B.workspace(size), scale=1.0)
    assert session.device_errors() == 0
    out, kv = out.cpu().double().view(rows, H, group, D), [tiles_sharp.held(c, b) for b in range(len(LENS))]
    for r, b, n in rows_of(LENS, new):
        if n <= 0:
            assert bool((out[r] == 0).all())
            continue
        p, v = tiles_sharp.answers(*kv[b], group, slice(0, n))
        assert float((out[r] - p @ v).abs().max()) <= tiles_sharp.bound(c, n), (r, b, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,H,group,page,win,sinks", [(64, 2, 1, 8, 40, 0), (128, 2, 4, 64, 30, 3), (128, 1, 16, 8, 70, 20), (256, 1, 3, 32, 9, 2)])
def test_windowed_tokens_keep_probabilities_in_two_parts(session, dtype, D, H, group, page, win, sinks):
    c = ref.Cache(LENS, H, D, page, dtype, seed=D + group)
    q = paged_sharp.fill(c, group, D + group).cuda()
    out = torch.full_like(q, 7.0)
    with ref.Buffers(session) as B:
        size = capi.paged_window_attention_workspace_bytes(len(LENS), len(LENS), H * group, H, D, c.slots, win, sinks)
        session.paged_window_attention(c.ids(B), B(q), B(out), H * group, win, sinks, workspace=B.workspace(size), scale=1.0)
    assert session.device_errors() == 0
    out = out.cpu().double().view(len(LENS), H, group, D)
    for b, n in enumerate(LENS):
        p, v = tiles_sharp.answers(*tiles_sharp.held(c, b), group, [s for s in range(n) if s >= n - win or s < sinks])
        assert float((out[b] - p @ v).abs().max()) <= paged_sharp.bound(c, b), (b, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,H,group,page", [(64, 2, 1, 8), (128, 2, 4, 16), (256, 1, 2, 16), (128, 1, 12, 32), (256, 1, 6, 8)])
def test_a_short_batch_behind_a_prefix_keeps_probabilities_in_two_parts(session, dtype, D, H, group, page):
    """The last sequence's pages are the prefix of the others."""
    c = ref.Cache(LENS, H, D, page, dtype, seed=D + group)
    tiles_sharp.fill(c, group, D + group)
    rows, length = len(LENS) - 1, LENS[-1]
    q = tiles_sharp.queries(c, group, rows).cuda()
    out = torch.full_like(q, 7.0)
    pages = c.table[-1, : -(-length // page)].contiguous()
    with ref.Buffers(session) as B:
        size = capi.paged_prefix_attention_workspace_bytes(rows, H * group, H, D, c.slots, pages.numel() * page)
        session.paged_prefix_attention(c.ids(B), B(pages), B(i32([length])), B(q), B(out), H * group, workspace=B.workspace(size), scale=1.0)
    assert session.device_errors() == 0
    out = out.cpu().double().view(rows, H, group, D)
    for b in range(rows):
        k, v = (torch.cat(both, 1) for both in zip(tiles_sharp.held(c, rows), tiles_sharp.held(c, b)))
        p, v = tiles_sharp.answers(k, v, group, slice(None))
        assert float((out[b] - p @ v).abs().max()) <= tiles_sharp.bound(c, length + LENS[b]), b
