"""Serving operators called by several host threads at once, a session and a
stream each."""
import threading

import pytest
import torch

from fercuda_b200 import capi
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu


class Caller(threading.Thread):
    """Calls an operator many times over buffers of its own."""

    def __init__(self, dim, grad, times, start):
        super().__init__()
        g = torch.Generator().manual_seed(dim)
        self.dim, self.grad, self.times, self.go, self.fault = dim, grad, times, start, None
        self.x, self.dy = (torch.randn(2500, 3 * dim, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
        self.pos = torch.randint(0, 5000, (2500, 1), generator=g, dtype=torch.int32).cuda()
        self.out = torch.zeros_like(self.x)
        torch.cuda.synchronize()

    def run(self):
        try:
            with capi.Session(0, pool_bytes=64 << 20) as s:
                b = [s.import_ptr(ref.CODES[t.dtype], list(t.shape), t.data_ptr()) for t in (self.x, self.dy, self.pos, self.out)]
                ws = s.alloc(capi.FER_DTYPE_U8, [capi.norm_rotary_grad_workspace_bytes(2500, 3, self.dim)])
                kw = dict(k_heads=1, sections=(self.dim // 2,))
                self.go.wait()
                for _ in range(self.times):
                    if self.grad:
                        job = s.norm_rotary_grad(b[0], b[1], b[3], b[2], 3, self.dim, workspace=ws, **kw)
                    else:
                        job = s.norm_rotary(b[0], b[3], b[2], 3, self.dim, **kw)
                s.wait(job)
                assert s.device_errors() == 0
        except BaseException as e:   # noqa: BLE001 - the main thread raises it
            self.fault = e


@pytest.mark.parametrize("grad", [False, True])
def test_two_threads_with_heads_of_different_sizes(grad):
    """One kernel, with shared memory by the size of the heads: what one call asks for does not go by the other."""
    start = threading.Barrier(2)
    callers = [Caller(dim, grad, 3000, start) for dim in (64, 128)]
    for c in callers:
        c.start()
    for c in callers:
        c.join()
    for c in callers:
        if c.fault:
            raise c.fault
    for c in callers:
        alone = Caller(c.dim, grad, 1, threading.Barrier(1))
        alone.run()
        assert alone.fault is None and ref.same_bits(c.out, alone.out)
