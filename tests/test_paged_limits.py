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
