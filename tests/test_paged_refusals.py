"""The native launchers of the rotary and paged-cache operators on the CPU:
what they refuse before any CUDA call, empty calls, workspace sizes, and the
ctypes mirrors of their structs."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

from fercuda_b200 import capi

ROOT = Path(__file__).resolve().parents[1]
OK, INVALID, NOT_SUPPORTED = 0, 1, 801   # cudaError_t
AT = 0x1000                              # an aligned address that is never used


def rotary(**change):
    a = dict(x=AT, out=2 * AT, positions=AT, x_stride=128, out_stride=128, rows=0, heads=2, head_dim=64, rotary_dim=64,
             axes=1, sections=(C.c_int * 4)(32), base=1e4, flags=0, dtype=capi.FER_DTYPE_BF16)
    a.update(change)
    return capi.kernels().fer_rotary(C.byref(capi.fer_rotary_args_t(**a)), None)


@pytest.mark.parametrize("change", [
    dict(x=None), dict(out=None), dict(positions=None), dict(rows=-1), dict(heads=0), dict(head_dim=0),
    dict(head_dim=63), dict(rotary_dim=0), dict(rotary_dim=31), dict(rotary_dim=66), dict(axes=0), dict(axes=5),
    dict(sections=(C.c_int * 4)(31)), dict(sections=(C.c_int * 4)(-1)), dict(axes=2, sections=(C.c_int * 4)(33, -1)),
    dict(base=0.0), dict(base=-1.0), dict(base=float("nan")), dict(base=float("inf")), dict(flags=8),
    dict(x_stride=127), dict(out_stride=127), dict(x=AT + 1), dict(out=AT, out_stride=256), dict(positions=AT + 2)])
def test_rotary_refuses(change):
    assert rotary(**change) == INVALID


@pytest.mark.parametrize("base", [1e-45, 3.1e38, 3.4028234e38])
def test_rotary_takes_every_finite_base(base):
    assert rotary(base=base) == OK


def test_rotary_takes_no_rows():
    assert rotary() == OK


def view(**change):
    v = dict(k=AT, v=2 * AT, page_table=AT, lengths=AT, batch=2, max_pages=4, pages=8, kv_heads=2, page_size=16,
             head_dim=64, dtype=capi.FER_DTYPE_F16)
    v.update(change)
    return capi.fer_paged_view_t(**v)


VIEWS = [(dict(k=None), INVALID), (dict(v=None), INVALID), (dict(page_table=None), INVALID),
         (dict(lengths=None), INVALID), (dict(batch=0), INVALID), (dict(max_pages=0), INVALID),
         (dict(pages=0), INVALID), (dict(kv_heads=0), INVALID), (dict(k=AT + 8), INVALID),
         (dict(page_table=AT + 2), INVALID), (dict(dtype=capi.FER_DTYPE_F32), NOT_SUPPORTED),
         (dict(head_dim=80), NOT_SUPPORTED), (dict(page_size=12), NOT_SUPPORTED), (dict(page_size=4), NOT_SUPPORTED),
         (dict(page_size=512), NOT_SUPPORTED), (dict(max_pages=1 << 28), NOT_SUPPORTED)]


def store(v=None, **change):
    a = dict(k_rows=AT, v_rows=AT, k_stride=128, v_stride=128, rows=0, n_seq=0, offsets=None, new_lengths=AT,
             weights=None, positions=None, seen=None, new_seen=None)
    a.update(change)
    return capi.kernels().fer_paged_store(C.byref(v or view()), C.byref(capi.fer_paged_store_args_t(**a)), None, None)


def attention(v=None, **change):
    a = dict(q=AT, out=2 * AT, q_stride=256, out_stride=256, n_seq=0, heads=4, scale=0.0, lse=None, weights=None,
             workspace=AT, workspace_bytes=1 << 30)
    a.update(change)
    return capi.kernels().fer_paged_attention(C.byref(v or view()), C.byref(capi.fer_paged_attention_args_t(**a)),
                                              None, None)


def evict(v=None, **change):
    a = dict(budget=8, recent=2, weights=AT, positions=AT, seen=AT, new_lengths=AT, new_weights=AT, new_positions=AT,
             workspace=AT, workspace_bytes=1 << 30)
    a.update(change)
    return capi.kernels().fer_paged_evict(C.byref(v or view()), C.byref(capi.fer_paged_evict_args_t(**a)), None, None)


@pytest.mark.parametrize("change,code", VIEWS)
def test_view_refused_by_every_operator(change, code):
    assert store(view(**change)) == attention(view(**change)) == evict(view(**change)) == code


@pytest.mark.parametrize("change", [
    dict(rows=-1), dict(n_seq=3), dict(n_seq=1), dict(rows=1), dict(new_lengths=None), dict(positions=AT),
    dict(positions=AT, seen=AT), dict(rows=1, n_seq=1, k_rows=None), dict(rows=1, n_seq=1, k_stride=127),
    dict(rows=1, n_seq=1, v_rows=AT + 1)])
def test_store_refuses(change):
    assert store(**change) == INVALID


@pytest.mark.parametrize("change", [
    dict(q=None), dict(out=None), dict(n_seq=3), dict(n_seq=-1), dict(heads=0), dict(heads=3), dict(q_stride=255),
    dict(out_stride=255), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=AT + 1),
    dict(n_seq=2, workspace=None), dict(n_seq=2, workspace=AT + 4), dict(n_seq=2, workspace_bytes=64)])
def test_attention_refuses(change):
    assert attention(**change) == INVALID


@pytest.mark.parametrize("change", [
    dict(budget=0), dict(recent=-1), dict(recent=9), dict(weights=None), dict(positions=None), dict(seen=None),
    dict(new_lengths=None), dict(new_weights=None), dict(new_positions=None), dict(workspace=None),
    dict(workspace=AT + 4), dict(workspace_bytes=8)])
def test_evict_refuses(change):
    assert evict(**change) == INVALID


@pytest.mark.parametrize("at", [AT + 1, AT + 2])
def test_misaligned_words_are_refused(at):
    """A kernel would fault on these addresses."""
    for name in ("offsets", "new_lengths", "weights", "seen", "new_seen"):
        assert store(**{name: at}) == INVALID, name
    assert store(positions=at, seen=AT, new_seen=AT) == store(positions=AT, seen=at, new_seen=AT) == INVALID
    assert store(positions=AT, seen=AT, new_seen=at) == INVALID
    for name in ("lse", "weights"):
        assert attention(**{name: at}) == INVALID, name
    for name in ("weights", "positions", "seen", "new_lengths", "new_weights", "new_positions"):
        assert evict(**{name: at}) == INVALID, name


@pytest.mark.parametrize("scale,code", [(2.5e38, INVALID), (3.0e38, INVALID), (2.0e38, OK), (1e-45, OK)])
def test_attention_takes_scales_with_a_finite_base_2_form(scale, code):
    """scale * log2 e is one f32 factor; were it infinite, a product of 0 would give NaN."""
    assert attention(scale=scale) == code


def test_no_sequences_is_no_work():
    assert store() == attention() == OK


def test_workspace_sizes():
    size = capi.paged_attention_workspace_bytes
    assert size(0, 4, 4, 64, 256) == size(1, 4, 4, 64, 0) == size(-1, 4, 4, 64, 256) == 0
    assert 0 < size(1, 4, 4, 64, 8) <= size(2, 4, 4, 64, 8) <= size(2, 4, 4, 128, 8)
    assert size(2, 8, 4, 64, 4096, True) >= size(2, 8, 4, 64, 4096) + 2 * 8 * 4096 * 4
    assert size(256, 64, 8, 128, 131072, True) > 1 << 32
    assert capi.paged_evict_workspace_bytes(4, 8, 1024, 100) >= 4 * 8 * 100 * 8
    assert capi.paged_evict_workspace_bytes(4, 8, 64, 100) > 0


def test_struct_layouts(tmp_path):
    names = ["fer_rotary_request_t", "fer_paged_cache_t", "fer_paged_store_request_t", "fer_paged_attention_request_t",
             "fer_paged_evict_request_t", "fer_rotary_args_t", "fer_paged_view_t", "fer_paged_store_args_t",
             "fer_paged_attention_args_t", "fer_paged_evict_args_t"]
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
    for name in ("fer_submit_rotary", "fer_submit_paged_store", "fer_submit_paged_attention",
                 "fer_submit_paged_evict"):
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
    assert s.rotary(1, 2, 3, 4, 64, sections=(5, 6, 7), rotary_dim=36, base=1e6, x_col=8, out_col=9, interleaved=True,
                    inverse=True) == 7
    want = capi.fer_rotary_request_t(1, 2, 3, 8, 9, 4, 64, 36, 3, (C.c_uint32 * 4)(5, 6, 7), 1e6, 5)
    assert got["fer_submit_rotary"] == bytes(want)
    s.paged_store(cache, 5, 6, k_col=7, v_col=8, offsets=9, new_lengths=10, weights=11, positions=12, seen=13, new_seen=14)
    want = capi.fer_paged_store_request_t(capi.fer_paged_cache_t(*cache), 5, 6, 9, 10, 11, 12, 13, 14, 7, 8)
    assert got["fer_submit_paged_store"] == bytes(want)
    s.paged_attention(cache, 5, 6, 7, workspace=8, q_col=9, out_col=10, scale=0.5, lse=11, weights=12)
    want = capi.fer_paged_attention_request_t(capi.fer_paged_cache_t(*cache), 5, 6, 11, 12, 8, 9, 10, 7, 0.5)
    assert got["fer_submit_paged_attention"] == bytes(want)
    s.paged_evict(cache, 5, 6, 7, 8, 9, workspace=10, new_lengths=11, new_weights=12, new_positions=13)
    want = capi.fer_paged_evict_request_t(capi.fer_paged_cache_t(*cache), 7, 8, 9, 11, 12, 13, 10, 5, 6)
    assert got["fer_submit_paged_evict"] == bytes(want)
