"""What the operators' cases leave behind in the session that they share, on the
CPU with a session that only counts."""
import gc

import torch

from fercuda_b200 import capi
from perf import operators


class Counting:
    def __init__(self):
        self.live, self.next = set(), 1

    def set_stream(self, handle):
        pass

    def import_ptr(self, dtype, shape, ptr):
        self.live.add(self.next)
        self.next += 1
        return self.next - 1

    def free(self, i):
        self.live.remove(i)


def test_a_state_frees_its_buffer_ids(monkeypatch):
    session = Counting()
    monkeypatch.setattr(operators, "_keep", {"session": session})
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: type("Stream", (), {"cuda_stream": 0}))
    monkeypatch.setattr(torch, "empty", lambda n, dtype, device: torch.zeros(16, dtype=dtype))
    monkeypatch.setattr(capi, "paged_attention_workspace_bytes", lambda *a: 16)
    case = next(c for c in operators.listed() if c["op"] == "attention")
    states = []
    for _ in range(3):
        s = dict(case=case, **{n: torch.zeros(1, dtype=torch.int32) for n in ("k", "v", "lengths", "q", "out", "lse")})
        s["table"] = torch.zeros(1, 7, dtype=torch.int32)
        operators._prepare_own(case, s)
        states.append(s)
    del s
    assert len(session.live) == 3 * 8    # seven tensors and the workspace each
    states.pop(0)
    gc.collect()
    assert len(session.live) == 2 * 8
    states.clear()
    gc.collect()
    assert not session.live
