"""The bound of tests/paged_sharp.py on the CPU: probabilities kept in two
16-bit parts meet it, and probabilities rounded once, or cut off, do not."""
import pytest
import torch

from tests import paged_ref as ref
from tests import paged_sharp as sharp


class HostCache:
    """What the bound needs of a ref.Cache, on the CPU: a page of 16 slots a sequence."""
    rows = ref.Cache.rows

    def __init__(self, lens, kv_heads, head_dim, dtype):
        self.lens, self.H, self.D, self.P, self.dtype = lens, kv_heads, head_dim, 16, dtype
        self.table = torch.arange(len(lens), dtype=torch.int32)[:, None]
        self.k = torch.full((len(lens), kv_heads, 16, head_dim), torch.nan, dtype=dtype)
        for b, n in enumerate(lens):
            self.k[b, :, :n] = 0
        self.v = self.k.clone()


def cut(p, dtype):
    """p to dtype, toward zero."""
    r = p.to(dtype)
    return torch.where(r.double() > p, torch.nextafter(r, torch.zeros_like(r)), r).double()


def kept(p, dtype, how):
    p = p / p.amax(-1, keepdim=True)     # as exp(s - max)
    if how == "rounded":
        return p.to(dtype).double()
    hi = cut(p, dtype)
    return hi if how == "cut" else hi + (p - hi).to(dtype).double()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,H,group,seed", [(64, 2, 1, 0), (128, 2, 4, 1), (256, 1, 16, 2)])
def test_bound_tells_two_parts_from_one(dtype, D, H, group, seed):
    c = HostCache([2, 3, 5, 8, 13, 16], H, D, dtype)
    sharp.fill(c, group, seed)
    off = {"two parts": [], "rounded": [], "cut": []}
    for b, (p, v) in enumerate(sharp.answers(c, group)):
        want = p @ v
        assert bool((want >= 1 - 1e-12).all()) and bool((want < 2).all())
        for how, worst in off.items():
            x = kept(p, dtype, how)
            total = (p / p.amax(-1, keepdim=True)).sum(-1, keepdim=True)
            worst.append(float(((x @ v / total).to(dtype).double() - want).abs().max()) / sharp.bound(c, b))
    assert max(off["two parts"]) <= 1.0
    assert max(off["rounded"]) > 1.0 and max(off["cut"]) > 1.0
    print(dtype, D, {k: round(max(v), 3) for k, v in off.items()})
