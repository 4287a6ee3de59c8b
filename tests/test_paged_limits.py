"""CPU suite: the paged cache's calls at the ends of their arguments' ranges -- what the host does before a launch, which without a GPU ends in an
error of the runtime's, and what is refused."""
import ctypes as C
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

from test_paged_refusals import ERR_ARG, PTR, attn, lib  # noqa: E402,F401

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(torch.cuda.is_available(), reason="the calls have no memory to work on: they must not reach a GPU")
@pytest.mark.parametrize("page", [1 << 30, (1 << 30) + 1, (1 << 31) - 1])
def test_one_page_of_more_than_2_30_rows(lib, page):  # noqa: F811
    """The call comes back (with the runtime's error): in a process of its own, which a host loop without an end would keep."""
    code = ("import ctypes as C, sys; sys.path[:0] = [%r, %r]; from test_paged_refusals import attn; from jukebox_amd import _lib as L; "
            "a = attn(n_pages=1, page_size=%d, max_pages=1); print(L.lib().jb_attn_paged(C.byref(a), None))" % (ROOT, os.path.join(ROOT, "tests"), page))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=60)
    assert r.stdout.strip() == "-3", r.stdout + r.stderr


def test_outputs_that_overlap_are_refused(lib):  # noqa: F811
    """Rows and heads that lie apart each, but not from one another; heads outside rows, and the single row or head whose stride is anything."""
    heads, D, T = 2, 128, 8
    for row, head, ok in ((256, 128, True), (128, 1024, True), (128, 128, False), (200, 128, False), (128, 200, False), (255, 128, False), (128, 1023, False), (1000, 500, True)):
        a = attn(out_row_stride=row, out_head_stride=head)
        rc = lib.jb_attn_paged_workspace(C.byref(a))
        assert (rc >= 0) == ok, (row, head)
        assert ok or b"overlap" in lib.jb_last_error()
    assert lib.jb_attn_paged_workspace(C.byref(attn(n_tokens=1, out_row_stride=128, out_head_stride=128))) >= 0
    assert lib.jb_attn_paged_workspace(C.byref(attn(n_head=1, n_kv_head=1, out_row_stride=128, out_head_stride=128))) >= 0


def test_pools_whose_rows_overlap_are_not_written(lib):  # noqa: F811
    from jukebox_amd import _lib as L

    def write(n_tokens=0, **kw):
        a = L.KvWriteArgs(L.F16, PTR, PTR, 256, 128, PTR, PTR, 4096, 256, 128, 10, 16, PTR, n_tokens, 2, 128)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.jb_kv_write(C.byref(a), None)

    assert write() == 0 and write(head_stride=2048, row_stride=128) == 0 and write(n_pages=1, page_stride=0) == 0
    assert write(n_kv_head=1, head_stride=0, row_stride=128) == 0 and write(page_size=1, row_stride=0) == 0
    # (a pool made by expand, heads inside one another, pages that share their last row)
    for kw in ({"page_stride": 0}, {"row_stride": 0}, {"head_stride": 64}, {"row_stride": 128}, {"page_stride": 4095}, {"head_stride": 2047, "row_stride": 128}):
        assert write(**kw) == ERR_ARG and b"overlap" in lib.jb_last_error(), kw


def test_more_pages_than_a_scan_counts(lib):  # noqa: F811
    from jukebox_amd import _lib as L
    for n, rc in (((1 << 30) + 1, -2), ((1 << 31) - 1, -2)):
        t, p = L.PageTable(PTR, 4, 3, 4, PTR, PTR, n, 1), L.PagePools((L.vp * 1)(PTR), 1, n, 512, 512)
        assert lib.jb_pages_fork(C.byref(t), C.byref(p), PTR, PTR, 0, PTR, PTR, None) == rc and b"2^30" in lib.jb_last_error()
        assert lib.jb_pages_compact(C.byref(t), C.byref(p), PTR + 16, PTR + 32, PTR, None) == rc and b"2^30" in lib.jb_last_error()
