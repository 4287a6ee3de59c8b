"""CPU suite: what the paged cache's operators and the filtered sampler refuse before anything is launched, at the C ABI and in the
Python layer, and the struct layouts they share with the header."""
import ctypes as C
import os
import subprocess

import pytest

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ERR_ARG, UNSUPPORTED = -1, -2


@pytest.fixture(scope="module")
def lib():
    from jukebox_amd import _lib as L
    from jukebox_amd.csrc.build import build
    build()
    return L.lib()


dummy = C.create_string_buffer(256)
PTR = (C.addressof(dummy) + 15) & ~15


def test_struct_layouts(tmp_path):
    from jukebox_amd import _lib as L
    pairs = [("jb_attn_paged_args", L.AttnPagedArgs), ("jb_kv_write_args", L.KvWriteArgs), ("jb_page_table", L.PageTable), ("jb_page_pools", L.PagePools),
             ("jb_sample_filtered_args", L.SampleFilteredArgs)]
    lines, expect = [], []
    for cname, ct in pairs:
        lines.append(f'printf("%zu\\n", sizeof({cname}));')
        expect.append(C.sizeof(ct))
        for fname, _ in ct._fields_:
            lines.append(f'printf("%zu\\n", offsetof({cname}, {fname}));')
            expect.append(getattr(ct, fname).offset)
    (tmp_path / "s.c").write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"jukebox_hip.h\"\nint main(void) {\n" + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")])
    assert [int(x) for x in subprocess.check_output([str(tmp_path / "s")]).split()] == expect


def attn(**kw):
    from jukebox_amd import _lib as L
    a = L.AttnPagedArgs(L.F16, 0, PTR, 256, 128, PTR, 256, 128, PTR, PTR, 4096, 256, 128, 10, 16, PTR, 4, 4, PTR, PTR, 8, 3, 2, 2, 128, 4, 64, 0, 0, 0.1, None, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc,word", [
    ({"dtype": 2}, ERR_ARG, b"dtype"), ({"attn_func": 6}, UNSUPPORTED, b"pages"), ({"attn_func": 7}, UNSUPPORTED, b"pages"), ({"attn_func": -1}, UNSUPPORTED, b"pages"),
    ({"n_head": 3}, ERR_ARG, b"dims"), ({"n_kv_head": 0}, ERR_ARG, b"dims"), ({"n_tokens": -1}, ERR_ARG, b"dims"), ({"d_head": 7}, UNSUPPORTED, b"8 to 512"),
    ({"d_head": 513}, UNSUPPORTED, b"8 to 512"), ({"n_pages": 0}, ERR_ARG, b"cache"), ({"page_size": 0}, ERR_ARG, b"cache"), ({"max_pages": 0}, ERR_ARG, b"cache"),
    ({"n_pages": 1 << 28, "page_size": 16}, ERR_ARG, b"2^31"), ({"row_stride": -1}, ERR_ARG, b"stride"), ({"out_row_stride": 0}, ERR_ARG, b"overlap"),
    ({"attn_func": 1}, ERR_ARG, b"block_ctx"), ({"window": -1}, ERR_ARG, b"window"), ({"attn_func": 1, "block_ctx": 4, "window": 4}, ERR_ARG, b"window"),
    ({"max_q": -1}, ERR_ARG, b"dims"), ({"q": None}, ERR_ARG, b"null"), ({"k": None}, ERR_ARG, b"null"), ({"out": None}, ERR_ARG, b"null"), ({"table": None}, ERR_ARG, b"null"),
    ({"lens": None}, ERR_ARG, b"null"), ({"cu_q": None}, ERR_ARG, b"null"),
    ({"max_len": 8192, "max_pages": 512}, ERR_ARG, b"workspace"), ({"max_len": 8192, "max_pages": 512, "workspace": PTR, "workspace_bytes": 64}, ERR_ARG, b"workspace")])
def test_attention_refuses(lib, kw, rc, word):
    a = attn(**kw)
    assert lib.jb_attn_paged(C.byref(a), None) == rc and word in lib.jb_last_error()
    if word not in (b"null", b"workspace"):
        assert lib.jb_attn_paged_workspace(C.byref(a)) == rc


def test_attention_of_nothing_and_workspace(lib):
    for kw in ({"n_tokens": 0}, {"n_seq": 0}, {"max_q": 0}):
        a = attn(q=None, out=None, **kw)
        assert lib.jb_attn_paged(C.byref(a), None) == 0 and lib.jb_attn_paged_workspace(C.byref(a)) == 0
    assert lib.jb_attn_paged(None, None) == ERR_ARG and lib.jb_attn_paged_workspace(None) == ERR_ARG
    assert lib.jb_attn_paged_workspace(C.byref(attn())) == 0                        # 64 tokens are not split
    need = lib.jb_attn_paged_workspace(C.byref(attn(max_len=8192, max_pages=512)))
    assert need > 0 and need % (8 * 2 * 4 * (128 + 2)) == 0                           # a state of 128 + 2 floats per row and split


def test_writes_and_pages_refuse(lib):
    from jukebox_amd import _lib as L

    def write(**kw):
        a = L.KvWriteArgs(L.F16, PTR, PTR, 256, 128, PTR, PTR, 4096, 256, 128, 10, 16, PTR, 8, 2, 128)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.jb_kv_write(C.byref(a), None)

    assert lib.jb_kv_write(None, None) == ERR_ARG
    for kw in ({"dtype": 2}, {"n_tokens": -1}, {"d_head": 0}, {"page_size": 0}, {"tok_stride": -1}, {"n_pages": 1 << 28}, {"k": None}, {"slots": None}, {"vpool": None}):
        assert write(**kw) == ERR_ARG, kw
    assert write(n_kv_head=1, d_head=7) == UNSUPPORTED and write(n_tokens=0, k=None) == 0

    def table(**kw):
        t = L.PageTable(PTR, 4, 3, 4, PTR, PTR, 10, 16)
        for k, v in kw.items():
            setattr(t, k, v)
        return C.byref(t)

    def pools(n=1, **kw):
        p = L.PagePools((L.vp * max(n, 1))(*([PTR] * n)), n, 10, 512, 512)
        for k, v in kw.items():
            setattr(p, k, v)
        return C.byref(p)

    null = L.PagePools((L.vp * 2)(PTR, None), 2, 10, 512, 512)
    for kw in ({"table": None}, {"lens": None}, {"ref": None}, {"n_seq": -1}, {"max_pages": 0}, {"n_pages": 0}, {"table_stride": 3}):
        assert lib.jb_pages_extend(table(**kw), PTR, 4, PTR, PTR, PTR, None) == ERR_ARG, kw
        assert lib.jb_pages_free(table(**kw), PTR, 1, PTR, None) == ERR_ARG, kw
        assert lib.jb_pages_fork(table(**kw), pools(), PTR, PTR, 1, PTR, PTR, None) == ERR_ARG, kw
        if "lens" not in kw:
            assert lib.jb_pages_compact(table(**kw), pools(), PTR + 16, PTR + 32, PTR, None) == ERR_ARG, kw
    assert lib.jb_pages_extend(table(page_size=0), PTR, 4, PTR, PTR, PTR, None) == ERR_ARG
    assert lib.jb_pages_extend(table(n_pages=1 << 21, page_size=1), PTR, 4, PTR, PTR, PTR, None) == UNSUPPORTED
    for bad in ((None, 4, PTR, PTR, PTR), (PTR, 4, None, PTR, PTR), (PTR, 4, PTR, None, PTR), (PTR, 4, PTR, PTR, None), (PTR, -1, PTR, PTR, PTR)):
        assert lib.jb_pages_extend(table(), *bad, None) == ERR_ARG
    assert lib.jb_pages_free(table(), PTR, 4, PTR, None) == ERR_ARG                    # more rows than the table has
    assert lib.jb_pages_free(table(n_seq=1 << 18), PTR, 4, PTR, None) == ERR_ARG
    assert lib.jb_pages_free(table(), None, 0, PTR, None) == 0
    assert lib.jb_pages_fork(table(), pools(), PTR, PTR, 4, PTR, PTR, None) == ERR_ARG
    assert lib.jb_pages_fork(table(n_pages=11), pools(), PTR, PTR, 1, PTR, PTR, None) == ERR_ARG
    assert lib.jb_pages_fork(table(), C.byref(null), PTR, PTR, 1, PTR, PTR, None) == ERR_ARG
    assert lib.jb_pages_fork(table(), pools(), PTR, PTR, 0, PTR, PTR, None) == 0
    assert lib.jb_pages_compact(table(), pools(), PTR, PTR + 32, PTR, None) == ERR_ARG     # the table itself
    for kw in ({"page_bytes": 0}, {"page_stride": 500}, {"n_pages": 0}, {"base": None}):
        assert lib.jb_pages_copy(pools(**kw), PTR, PTR, 1, None) == ERR_ARG, kw
    assert lib.jb_pages_copy(pools(), None, PTR, 1, None) == ERR_ARG and lib.jb_pages_copy(pools(), None, None, 0, None) == 0


def test_sampler_refuses(lib):
    from jukebox_amd import _lib as L

    def call(**kw):
        a = L.SampleFilteredArgs(L.F32, PTR, 100, 4, 100, PTR, None, None, None, None, 1.0, 0, 0.0, 0.0, PTR)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.jb_sample_filtered(C.byref(a), None)

    assert lib.jb_sample_filtered(None, None) == ERR_ARG
    for kw in ({"dtype": 2}, {"bins": 0}, {"rows": -1}, {"ld": 99}, {"logits": None}, {"u": None}, {"tokens": None}):
        assert call(**kw) == ERR_ARG, kw
    assert call(bins=262145, ld=262145) == UNSUPPORTED and call(rows=0, logits=None) == 0


def test_python_layer_refuses_wrong_tensors(lib):
    from jukebox_amd import hip_ops as H
    from jukebox_amd._lib import JukeboxHipError
    f = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    for call in (lambda: H.attn_paged(f(2, 2, 64), f(4, 16, 2, 64), f(4, 16, 2, 64), i(1, 4), i(1), i(2)),                     # not on a GPU
                 lambda: H.attn_paged(f(2, 2, 64).double(), f(4, 16, 2, 64), f(4, 16, 2, 64), i(1, 4), i(1), i(2)),            # type
                 lambda: H.attn_paged(f(2, 2, 64), f(4, 16, 2, 64).float(), f(4, 16, 2, 64), i(1, 4), i(1), i(2)),
                 lambda: H.kv_write(f(2, 2, 64), f(2, 2, 64), f(4, 16, 2, 64), f(4, 16, 2, 64), torch.zeros(2, dtype=torch.int64)),
                 lambda: H.pages_extend(i(2, 4), i(2), i(9), i(3), 16, 3, i(1)),
                 lambda: H.pages_extend(i(2, 4).long(), i(2), i(9), i(3), 16, 3, i(1)),
                 lambda: H.pages_extend(i(4, 2).T, i(2), i(9), i(3), 16, 3, i(1)),
                 lambda: H.pages_free(i(2, 4), i(3), i(9), i(1), i(1)),
                 lambda: H.pages_fork([f(9, 16, 8)], i(2, 4), i(2), i(9), i(1), i(1), 16, i(1)),
                 lambda: H.pages_compact([f(9, 16, 8)], i(2, 4), i(9)),
                 lambda: H.pages_copy([f(9, 16, 8)], i(1), i(1)),
                 lambda: H.pages_copy([f(9, 16, 8), f(9, 16, 9)], i(1), i(1)),
                 lambda: H.pages_copy([f(9, 8, 16).transpose(1, 2)], i(1), i(1)),
                 lambda: H.sample_filtered(f(2, 8), torch.zeros(2)), lambda: H.sample_filtered(f(2, 8), 0.5), lambda: H.sample_filtered(f(8), torch.zeros(8)),
                 lambda: H.sample_filtered(f(2, 8), torch.zeros(2), temp=torch.zeros(3)), lambda: H.sample_filtered(f(2, 8), torch.zeros(2), top_k=torch.zeros(2)),
                 lambda: H.sample_filtered(torch.zeros(2, 8, dtype=torch.int32), torch.zeros(2))):
        with pytest.raises(JukeboxHipError):
            call()
    assert H.pages_copy([], i(0), i(0)) is None


@pytest.mark.parametrize("n_tokens,max_q,d_head", [(65536, 1, 128), (65536, 1, 512), (400000, 1, 64), (1 << 22, 4, 128), (65536, 300, 128)])
def test_workspace_of_a_padded_batch(lib, n_tokens, max_q, d_head):
    """Four sequences in buffers of many more rows: the split states take 1 GiB at most."""
    need = lib.jb_attn_paged_workspace(C.byref(attn(n_tokens=n_tokens, n_seq=4, n_head=32, n_kv_head=8, d_head=d_head, q_row_stride=32 * d_head,
                                                    out_row_stride=32 * d_head, q_head_stride=d_head, out_head_stride=d_head, max_q=max_q,
                                                    max_len=131072, max_pages=8192)))
    assert 0 <= need <= 1 << 30
