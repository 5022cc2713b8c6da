"""The native launchers of the serving step's operators on the CPU: what they
refuse before any CUDA call, empty calls, workspace sizes, and the ctypes
mirrors of their structs."""
import ctypes as C
import subprocess

import pytest

from fercuda_b200 import capi
from tests.test_paged_refusals import AT, INVALID, NOT_SUPPORTED, OK, ROOT, VIEWS, view


def norm_args(**change):
    a = dict(x=AT, out=2 * AT, positions=AT, x_stride=128, out_stride=128, rows=0, heads=2, head_dim=64, rotary_dim=64,
             axes=1, sections=(C.c_int * 4)(32), base=1e4, flags=0, dtype=capi.FER_DTYPE_BF16)
    n = dict(k_heads=1, q_gamma=AT, k_gamma=AT, eps=1e-6)
    n.update({k: change.pop(k) for k in list(change) if k in n})
    a.update(change)
    return capi.fer_norm_rotary_args_t(capi.fer_rotary_args_t(**a), **n)


def norm(**change):
    return capi.kernels().fer_norm_rotary(C.byref(norm_args(**change)), None, None)


def norm_grad(**change):
    d = dict(grad=3 * AT, grad_stride=128, q_gamma_grad=None, k_gamma_grad=None, workspace=AT, workspace_bytes=1 << 20)
    d.update({k: change.pop(k) for k in list(change) if k in d})
    return capi.kernels().fer_norm_rotary_grad(C.byref(norm_args(**change)), C.byref(capi.fer_norm_rotary_grad_t(**d)), None, None)


@pytest.mark.parametrize("change", [
    dict(x=None), dict(out=None), dict(positions=None), dict(rows=-1), dict(heads=0), dict(heads=65537), dict(head_dim=0), dict(head_dim=63),
    dict(head_dim=258, x_stride=600, out_stride=600), dict(rotary_dim=0), dict(rotary_dim=31), dict(rotary_dim=66), dict(axes=0),
    dict(axes=5), dict(sections=(C.c_int * 4)(31)), dict(axes=2, sections=(C.c_int * 4)(33, -1)), dict(base=0.0), dict(base=float("nan")),
    dict(base=float("inf")), dict(flags=4), dict(flags=8), dict(x_stride=127), dict(out_stride=127), dict(x=AT + 1),
    dict(out=AT, out_stride=256), dict(positions=AT + 2), dict(k_heads=-1), dict(k_heads=3), dict(eps=-1e-9), dict(eps=float("nan")),
    dict(eps=float("inf")), dict(q_gamma=AT + 2), dict(k_gamma=AT + 1)])
def test_norm_rotary_refuses(change):
    assert norm(**dict(change)) == INVALID
    assert norm_grad(**dict(change)) == INVALID


@pytest.mark.parametrize("change", [
    dict(grad=None), dict(grad_stride=127), dict(grad=AT + 1), dict(q_gamma_grad=AT + 2), dict(k_gamma_grad=AT + 1),
    dict(workspace=None), dict(workspace=AT + 8), dict(workspace_bytes=8), dict(out=3 * AT, out_stride=256)])
def test_norm_rotary_grad_refuses(change):
    assert norm_grad(**change) == INVALID


def test_norm_rotary_takes_no_rows_and_no_gammas():
    assert norm() == norm(q_gamma=None, k_gamma=None) == norm(eps=0.0) == norm(k_heads=0) == norm(k_heads=2) == norm_grad() == OK
    assert norm(dtype=4) == norm_grad(dtype=4) == NOT_SUPPORTED


PLAN = ("page_table", "lengths", "counts", "held", "seen", "free_pages", "free_state", "new_held", "new_free_state", "offsets",
        "sequences", "positions", "slots")


def plan(**change):
    a = {n: AT for n in PLAN}
    a.update(batch=2, max_pages=4, pages=8, page_size=16, rows=4)
    a.update(change)
    return capi.kernels().fer_paged_plan(C.byref(capi.fer_paged_plan_args_t(**a)), None, None)


@pytest.mark.parametrize("name", PLAN)
def test_plan_refuses_addresses(name):
    if name not in ("seen", "sequences", "positions", "slots"):
        assert plan(**{name: None}) == INVALID
    assert plan(**{name: AT + 1}) == plan(**{name: AT + 2}) == INVALID


@pytest.mark.parametrize("change,code", [
    (dict(batch=0), INVALID), (dict(max_pages=0), INVALID), (dict(pages=0), INVALID), (dict(rows=-1), INVALID),
    (dict(page_size=12), NOT_SUPPORTED), (dict(page_size=4), NOT_SUPPORTED), (dict(page_size=512), NOT_SUPPORTED),
    (dict(batch=65536), NOT_SUPPORTED), (dict(max_pages=1 << 27), NOT_SUPPORTED), (dict(pages=1 << 27), NOT_SUPPORTED)])
def test_plan_refuses(change, code):
    assert plan(**change) == code


def window(v=None, **change):
    a = dict(q=AT, out=2 * AT, q_stride=256, out_stride=256, rows=0, n_seq=0, heads=4, offsets=None, window=0, sinks=0, scale=0.0,
             lse=None, workspace=AT, workspace_bytes=1 << 30)
    a.update(change)
    return capi.kernels().fer_paged_window_attention(C.byref(v or view()), C.byref(capi.fer_paged_window_args_t(**a)), None, None)


def prefix(v=None, **change):
    a = dict(q=AT, out=2 * AT, q_stride=256, out_stride=256, n_seq=0, heads=4, prefix_pages=AT, prefix_length=AT, max_prefix_pages=2,
             scale=0.0, lse=None, workspace=AT, workspace_bytes=1 << 30)
    a.update(change)
    return capi.kernels().fer_paged_prefix_attention(C.byref(v or view()), C.byref(capi.fer_paged_prefix_args_t(**a)), None, None)


@pytest.mark.parametrize("change,code", VIEWS)
def test_view_refused(change, code):
    assert window(view(**change)) == prefix(view(**change)) == code


SHARED = [dict(q=None), dict(out=None), dict(n_seq=3, rows=3), dict(n_seq=-1), dict(heads=0), dict(heads=3), dict(q_stride=255),
          dict(out_stride=255), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3.0e38), dict(q=AT + 1),
          dict(out=AT + 1), dict(lse=AT + 2)]


@pytest.mark.parametrize("change", SHARED + [
    dict(rows=-1), dict(n_seq=1), dict(rows=2, n_seq=1), dict(offsets=AT + 2), dict(window=-1), dict(sinks=-1),
    dict(offsets=AT, rows=5, n_seq=3)])
def test_window_attention_refuses(change):
    assert window(**change) == INVALID


@pytest.mark.parametrize("change", SHARED + [
    dict(prefix_pages=None), dict(prefix_length=None), dict(prefix_pages=AT + 2), dict(prefix_length=AT + 1), dict(max_prefix_pages=-1)])
def test_prefix_attention_refuses(change):
    change = {k: v for k, v in change.items() if k != "rows"}
    assert prefix(**change) == INVALID


@pytest.mark.parametrize("change", [dict(workspace=None), dict(workspace=AT + 4), dict(workspace_bytes=16)])
def test_workspaces_are_refused(change):
    long = view(max_pages=1 << 12)      # split over the keys
    assert capi.paged_window_attention_workspace_bytes(2, 2, 4, 2, 64, 16 << 12, 0, 0) > 16
    assert window(long, n_seq=2, rows=2, **change) == prefix(long, n_seq=2, **change) == INVALID


def test_no_sequences_is_no_work():
    assert window() == window(offsets=AT) == window(scale=1e-45) == prefix() == OK


def test_workspace_sizes():
    size = capi.norm_rotary_grad_workspace_bytes
    assert 0 < size(0, 4, 64) <= size(1, 4, 64) <= size(1000, 4, 64) <= size(1000, 4, 256)
    assert size(2 ** 31 - 1, 65536, 256) < 1 << 21      # partial sums of a bounded number of CTAs
    size = capi.paged_window_attention_workspace_bytes
    assert size(1, 1, 4, 4, 64, 256, 0, 0) > 0
    assert size(2, 2, 8, 4, 64, 4096, 0, 0) >= size(1, 1, 8, 4, 64, 4096, 0, 0)
    assert size(0, 0, 4, 4, 64, 256, 0, 0) >= 0 and size(1 << 20, 4096, 64, 8, 128, 1 << 20, 4096, 4) < 1 << 34
    size = capi.paged_prefix_attention_workspace_bytes
    assert size(1, 4, 4, 64, 256, 64) > 0
    assert size(64, 32, 8, 128, 1024, 8192) >= size(4, 32, 8, 128, 1024, 8192)


def test_struct_layouts(tmp_path):
    names = ["fer_norm_rotary_request_t", "fer_norm_rotary_grad_request_t", "fer_paged_plan_request_t",
             "fer_paged_window_attention_request_t", "fer_paged_prefix_attention_request_t", "fer_norm_rotary_args_t",
             "fer_norm_rotary_grad_t", "fer_paged_plan_args_t", "fer_paged_window_args_t", "fer_paged_prefix_args_t"]
    lines = []
    for n in names:
        lines.append(f'printf("{n} %zu\\n", sizeof({n}));')
        lines += [f'printf("{n}.{f[0]} %zu\\n", offsetof({n}, {f[0]}));' for f in getattr(capi, n)._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "fercuda/b200/ext.h"\n'
                   '#include "fercuda/b200/native.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT}/include", "-I/usr/local/cuda/include", str(src), "-o",
                    str(tmp_path / "probe")], check=True)
    got = dict(line.split() for line in subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True,
                                                       check=True).stdout.splitlines())
    for n in names:
        t = getattr(capi, n)
        assert int(got[n]) == C.sizeof(t), n
        for f in t._fields_:
            assert int(got[f"{n}.{f[0]}"]) == getattr(t, f[0]).offset, (n, f[0])


def test_session_entries_refuse_null():
    lib = capi.capi()
    for name in ("fer_submit_norm_rotary", "fer_submit_norm_rotary_grad", "fer_submit_paged_plan", "fer_submit_paged_window_attention",
                 "fer_submit_paged_prefix_attention"):
        assert getattr(lib, name)(None, None, None).code == capi.FER_STATUS_INVALID_ARGUMENT


def test_packed_requests_are_the_structs():
    """The bytes that Session packs for a call are those of the ctypes mirror with the same values."""
    got = {}

    class Fake:
        def __getattr__(self, name):
            def fn(ptr, request, job):
                got[name] = request
                return capi.fer_status_t(0, None)
            return fn

    s = capi.Session.__new__(capi.Session)
    s.lib, s.ptr, s._job, s._job_ref = Fake(), None, C.c_uint64(7), None
    cache = capi.paged_cache(1, 2, 3, 4)
    box = capi.fer_paged_cache_t(*cache)
    turn = capi.fer_rotary_request_t(1, 2, 3, 8, 9, 4, 64, 36, 3, (C.c_uint32 * 4)(5, 6, 7), 1e6, 1)
    kw = dict(sections=(5, 6, 7), rotary_dim=36, base=1e6, x_col=8, out_col=9, interleaved=True, k_heads=10, q_gamma=11, k_gamma=12,
              eps=0.25)
    assert s.norm_rotary(1, 2, 3, 4, 64, **kw) == 7
    assert got["fer_submit_norm_rotary"] == bytes(capi.fer_norm_rotary_request_t(turn, 11, 12, 10, 0.25))
    s.norm_rotary_grad(1, 13, 2, 3, 4, 64, workspace=14, q_gamma_grad=15, k_gamma_grad=16, grad_col=17, **kw)
    want = capi.fer_norm_rotary_grad_request_t(turn, 11, 12, 13, 15, 16, 14, 17, 10, 0.25, 0)
    assert got["fer_submit_norm_rotary_grad"] == bytes(want)
    s.paged_plan(1, 2, 3, 4, 5, 6, 7, page_size=8, new_held=9, new_free_state=10, sequences=11, positions=12, slots=13, seen=14)
    want = capi.fer_paged_plan_request_t(1, 2, 3, 4, 5, 6, 7, 9, 10, 11, 12, 13, 14, 8, 0)
    assert got["fer_submit_paged_plan"] == bytes(want)
    s.paged_window_attention(cache, 5, 6, 7, 8, 9, workspace=10, offsets=11, q_col=12, out_col=13, scale=0.5, lse=14)
    want = capi.fer_paged_window_attention_request_t(box, 5, 6, 14, 11, 10, 12, 13, 7, 8, 9, 0.5)
    assert got["fer_submit_paged_window_attention"] == bytes(want)
    s.paged_prefix_attention(cache, 5, 6, 7, 8, 9, workspace=10, q_col=11, out_col=12, scale=0.5, lse=13)
    want = capi.fer_paged_prefix_attention_request_t(box, 7, 8, 13, 5, 6, 10, 11, 12, 9, 0.5)
    assert got["fer_submit_paged_prefix_attention"] == bytes(want)
    for call in (s.norm_rotary, s.norm_rotary_grad):
        with pytest.raises(ValueError):
            call(*([1, 2, 3, 4, 64] if call == s.norm_rotary else [1, 13, 2, 3, 4, 64]), sections=(1, 2, 3, 4, 5),
                 **({} if call == s.norm_rotary else dict(workspace=1)))
