"""The bound of tests/tiles_sharp.py on the CPU, at the sizes that the GPU tests
have: probabilities rounded to nearest in two 16-bit parts meet it, and rounded
once they do not."""
import pytest
import torch

from tests import tiles_sharp
from tests.test_gpu_tiles_sharp import LENS, SHAPES, rows_of
from tests.test_paged_sharp_bound import HostCache


class HostPages(HostCache):
    def __init__(self, lens, kv_heads, head_dim, dtype):
        super().__init__(lens, kv_heads, head_dim, dtype)
        self.P = max(lens)
        self.k = torch.full((len(lens), kv_heads, self.P, head_dim), torch.nan, dtype=dtype)
        for b, n in enumerate(lens):
            self.k[b, :, :n] = 0
        self.v = self.k.clone()


def kept(p, dtype, parts):
    up = 256.0 if dtype == torch.float16 else 1.0
    p = p / p.amax(-1, keepdim=True) * up
    hi = p.to(dtype).double()
    return (hi + (p - hi).to(dtype).double() if parts == 2 else hi) / up


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,H,group,page,new", SHAPES)
def test_bound_tells_two_parts_from_one(dtype, D, H, group, page, new):
    c = HostPages(LENS, H, D, dtype)
    tiles_sharp.fill(c, group, D + group)
    off, kv = {1: 0.0, 2: 0.0}, [tiles_sharp.held(c, b) for b in range(len(LENS))]
    for _, b, n in rows_of(LENS, new):
        if n <= 0:
            continue
        p, v = tiles_sharp.answers(*kv[b], group, slice(0, n))
        want, total = p @ v, (p / p.amax(-1, keepdim=True)).sum(-1, keepdim=True)
        assert bool((want >= 1 - 1e-12).all()) and bool((want < 2).all())
        for parts in off:
            got = (kept(p, dtype, parts) @ v / total).to(dtype).double()
            off[parts] = max(off[parts], float((got - want).abs().max()) / tiles_sharp.bound(c, n))
    assert off[2] <= 1.0 < off[1], off
