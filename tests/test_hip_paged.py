"""GPU suite: the paged key / value cache -- attention over pages, writes into them, the control of the pages -- against the
operators' definitions in 64 bits.

Tolerance of an attention output, element by element (u = half a step of the output's type, relative):
    |got - want| <= u |want| + (2 ds + dp + n 2^-24) sum_k p_k |v_k| + tiny
  ds  error of a score: D products summed in fp32, at most D 2^-24 sum_d |q_d k_d| scale, and two roundings of the scaled score;
      p changes by the factor exp(+-ds) and its normalisation by another
  dp  the probabilities enter the products in two parts of the 16-bit type: 2^-16 (bfloat16), 2^-22 (half); the chunk kernel's
      enter rounded once: 2^-8, 2^-11; plus 2^-22 for the exponential
  n   fp32 additions that a product's accumulator goes through one after the other: keys / 64 + 64 covers every kernel's order
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DENSE, BLOCK, TRANSPOSE, PREV = 0, 1, 2, 3
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def H():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from jukebox_amd import _lib, hip_ops
    _lib.lib()          # fail loudly if the extension is missing
    return hip_ops


def visible(func, bc, window, qpos, kpos):
    if func == BLOCK:
        return (kpos <= qpos) & (kpos // bc == qpos // bc)
    if func == TRANSPOSE:
        return (kpos <= qpos) & ((qpos - kpos) % bc == 0)
    if func == PREV:
        return kpos // bc == qpos // bc - 1
    return (kpos <= qpos) & ((kpos > qpos - window) if window else (kpos >= 0))


class Batch:
    """A ragged batch on pages that lie anywhere: lens[i] tokens, the last nq[i] of them queries.  What no query may read --
    rows behind a sequence's end, pages of nobody -- is NaN."""

    def __init__(self, dtype, lens, nq, heads, kv, D, page, seed=0, spare=2, layout="nhd", gap=0):
        g = torch.Generator("cuda").manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.dtype, self.lens, self.nq, self.page, self.D, self.kv, self.heads = dtype, lens, nq, page, D, kv, heads
        need = [-(-n // page) for n in lens]
        P, width = sum(need) + spare, max(need + [1]) + 1
        order = rng.permutation(P)
        table = np.full((len(lens), width), -1, np.int32)
        shape = (P, kv, page, D) if layout == "hnd" else (P, page, kv, D)
        # `gap` channels lie between two rows, so that strides are not those of a packed cache
        store = torch.full((2,) + shape[:3] + (D + gap,), math.nan, device="cuda", dtype=dtype)
        if layout == "hnd":
            store = store.transpose(2, 3)
        self.k, self.v = store[0, ..., :D], store[1, ..., :D]
        at = 0
        for i, n in enumerate(lens):
            table[i, :need[i]] = order[at:at + need[i]]
            at += need[i]
        self.table = torch.from_numpy(table).cuda()
        self.rows_k, self.rows_v = [], []
        for i, n in enumerate(lens):
            kk = torch.randn(n, kv, D, generator=g, device="cuda").to(dtype)
            vv = torch.randn(n, kv, D, generator=g, device="cuda").to(dtype)
            pos = torch.arange(n, device="cuda")
            pg = self.table[i, (pos // page)].long() if n else pos
            self.k[pg, pos % page], self.v[pg, pos % page] = kk, vv
            self.rows_k.append(kk.double())
            self.rows_v.append(vv.double())
        self.cu = torch.tensor(np.concatenate([[0], np.cumsum(nq)]), dtype=torch.int32, device="cuda")
        self.len_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.q = torch.randn(sum(nq), heads, D, generator=g, device="cuda").to(dtype)

    def want(self, func=DENSE, bc=0, window=0, scale=None, blind=None):
        """(values, tolerances) in 64 bits.  blind(i, positions) -> positions of sequence i that no page holds."""
        scale = 1.0 / math.sqrt(self.D) if scale is None else scale
        u = torch.finfo(self.dtype).eps / 2
        dp = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[self.dtype] + 2.0 ** -22
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        tol = torch.full_like(out, 1e-30)
        at = 0
        for i, (n, nq) in enumerate(zip(self.lens, self.nq)):
            q = self.q[at:at + nq].double()
            kpos, qpos = torch.arange(n, device="cuda"), torch.arange(n - nq, n, device="cuda")
            see = visible(func, bc, window, qpos[:, None], kpos[None, :])
            if blind is not None and n:
                see &= ~blind(i, kpos)[None, :]
            for h in range(self.heads):
                j = h * self.kv // self.heads
                k = torch.where(see.any(0)[:, None], self.rows_k[i][:, j], 0.0)
                v = torch.where(see.any(0)[:, None], self.rows_v[i][:, j], 0.0)
                s = torch.where(see, (q[:, h] @ k.T) * scale, -math.inf)
                ds = self.D * 2.0 ** -24 * (q[:, h].abs() @ k.abs().T) * abs(scale) + 3 * 2.0 ** -24 * torch.where(see, s.abs(), 0.0)
                p = torch.where(see, torch.softmax(s, 1), 0.0) if n else s
                o = p @ v
                e = (2 * ds.amax(1, keepdim=True) + dp + (n / 64 + 64) * 2.0 ** -24) if n else torch.zeros(nq, 1, device="cuda")
                out[at:at + nq, h] = o
                tol[at:at + nq, h] += u * o.abs() + e * (p @ v.abs()) * (1 + u) + (2.0 ** -24 if self.dtype == torch.float16 else 0.0)
            at += nq
        return out, tol

    def run(self, H, **kw):
        return H.attn_paged(self.q, self.k, self.v, self.table, self.len_t, self.cu, **kw)

    def check(self, H, func=DENSE, bc=0, window=0, scale=None, **kw):
        got = self.run(H, func=func, block_ctx=bc, window=window, scale=scale, **kw)
        torch.cuda.synchronize()
        want, tol = self.want(func, bc, window, scale)
        off = (got.double() - want).abs()
        assert bool((off <= tol).all()), f"off by {float((off / tol).max()):.3g} tolerances, {int((~(off <= tol)).sum())} of {off.numel()} elements"
        return got


ONE = [("one", [1], [1]), ("few", [5, 33, 1, 64], [1, 1, 1, 1]), ("long", [1500, 7, 4097], [1, 1, 1]), ("idle", [40, 0, 17], [1, 0, 1])]
CHUNK = [("whole", [70, 1, 33], [70, 1, 33]), ("tail", [300, 129, 64], [37, 128, 2]), ("mixed", [513, 40, 0, 9], [200, 0, 0, 9])]
HEADS = [(1, 1, 480), (2, 2, 256), (8, 8, 150), (8, 2, 128), (4, 4, 64), (6, 2, 80), (5, 5, 33), (8, 1, 8), (2, 1, 512), (40, 2, 17)]


@pytest.mark.parametrize("dt", sorted(TYPES))
@pytest.mark.parametrize("heads,kv,D", HEADS)
@pytest.mark.parametrize("name,lens,nq", ONE + CHUNK, ids=[c[0] for c in ONE + CHUNK])
def test_attention_over_pages(H, dt, heads, kv, D, name, lens, nq):
    page = {"one": 16, "few": 7, "long": 64, "idle": 1, "whole": 20, "tail": 48, "mixed": 128}[name]
    Batch(TYPES[dt], lens, nq, heads, kv, D, page, seed=D + heads).check(H)


@pytest.mark.parametrize("dt", sorted(TYPES))
@pytest.mark.parametrize("func,bc,window", [(DENSE, 0, 1), (DENSE, 0, 50), (DENSE, 0, 100000), (BLOCK, 32, 0), (BLOCK, 7, 0), (PREV, 32, 0), (PREV, 100, 0),
                                            (TRANSPOSE, 32, 0), (TRANSPOSE, 5, 0), (TRANSPOSE, 1000, 0), (BLOCK, 1, 0), (PREV, 1, 0), (TRANSPOSE, 1, 0)])
@pytest.mark.parametrize("nq", [[1, 1, 1], [150, 31, 1], [600, 65, 3]], ids=["one", "chunk", "whole"])
def test_patterns(H, dt, func, bc, window, nq):
    for heads, kv, D in [(2, 2, 64), (6, 2, 150)]:
        Batch(TYPES[dt], [600, 65, 3], nq, heads, kv, D, 24, seed=bc + window).check(H, func, bc, window)


def test_patterns_agree_with_the_fixed_cache(H):
    """The same rows in a cache of fixed length per sample: the framework's prefill attention, every pattern that pages hold."""
    N, n, nq, heads, D, bc, page = 3, 200, 77, 2, 48, 32, 16
    b = Batch(torch.float32, [n] * N, [nq] * N, heads, heads, D, page, seed=5)
    k = torch.stack([r.float().reshape(n, heads * D) for r in b.rows_k]).contiguous()
    v = torch.stack([r.float().reshape(n, heads * D) for r in b.rows_v]).contiguous()
    for func in (DENSE, BLOCK, TRANSPOSE, PREV):
        got = b.run(H, func=func, block_ctx=bc).reshape(N, nq, heads * D)
        want = H.attn_prefill(func, b.q.reshape(N, nq, heads * D).contiguous(), k, v, heads, bc, n - nq)
        # two fp32 evaluations of the same sums
        assert float((got - want).abs().max()) < 2e-5


@pytest.mark.parametrize("dt", sorted(TYPES))
@pytest.mark.parametrize("layout,gap", [("hnd", 0), ("nhd", 3), ("hnd", 8)])
def test_strides_and_layouts(H, dt, layout, gap):
    for heads, kv, D in [(4, 2, 128), (3, 3, 50)]:
        b = Batch(TYPES[dt], [130, 31, 2], [40, 1, 2], heads, kv, D, 16, seed=gap, layout=layout, gap=gap)
        b.check(H)
        # queries and outputs that are parts of larger tensors
        want = b.run(H)
        wide = torch.randn(sum(b.nq), 3 * heads, D + 5, device="cuda").to(b.dtype)
        wide[:, heads:2 * heads, 2:D + 2] = b.q
        q = wide[:, heads:2 * heads, 2:D + 2]
        hold = torch.zeros(heads, sum(b.nq), D + 1, device="cuda", dtype=b.dtype)
        got = H.attn_paged(q, b.k, b.v, b.table, b.len_t, b.cu, out=hold.transpose(0, 1)[..., :D])
        assert torch.equal(got, want)
        assert float(hold[..., D:].abs().max()) == 0.0


@pytest.mark.parametrize("dt", sorted(TYPES))
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_masked_keys_and_values_may_hold_anything(H, dt, what):
    """NaN and infinity in the rows of LATER positions of the chunk reach only the queries that see them."""
    for heads, kv, D, lens, nq in [(2, 2, 64, [100], [60]), (2, 1, 256, [40, 70], [40, 3]), (1, 1, 480, [50], [17]), (4, 2, 150, [300], [130])]:
        b = Batch(TYPES[dt], lens, nq, heads, kv, D, 16, seed=3)
        clean, _ = b.want()
        ref = b.run(H)
        for i, n in enumerate(lens):
            pos = n - 2                                     # the last but one: seen by the last two queries only
            pg = int(b.table[i, pos // 16])
            b.v[pg, pos % 16, :, D // 3] = what
            b.k[pg, pos % 16, 0, 1] = math.nan
        got = b.run(H)
        at = 0
        for i, c in enumerate(nq):
            rows = slice(at, at + c - 2)
            assert torch.equal(got[rows], ref[rows])
            assert not torch.isfinite(got[at + c - 1].float()).all()
            at += c


def test_pages_that_do_not_exist_are_masked(H):
    b = Batch(torch.bfloat16, [100, 64], [30, 1], 4, 2, 64, 16, seed=8)
    table = b.table.clone()
    table[0, 2], table[1, 0], table[1, 3] = -1, 10 ** 6, b.k.shape[0]
    b.table = table

    def blind(i, pos):
        p = pos // 16
        return (p == 2) if i == 0 else (p == 0) | (p == 3)

    got = b.run(H)
    want, tol = b.want(blind=blind)
    assert bool(((got.double() - want).abs() <= tol).all())
    b.table = torch.full_like(table, -1)
    assert float(b.run(H).float().abs().max()) == 0.0


def test_lengths_that_do_not_fit_are_clamped(H):
    """A length beyond the table's pages, a negative one, one shorter than the chunk: no access outside, zeros where no key is."""
    b = Batch(torch.float16, [48, 48, 48], [10, 10, 10], 2, 2, 64, 16, seed=9)
    ref = b.run(H)
    lens = torch.tensor([10 ** 9, -5, 4], dtype=torch.int32, device="cuda")
    table = b.table[:, :3].contiguous()
    got = H.attn_paged(b.q, b.k, b.v, table, lens, b.cu)
    assert torch.equal(got[:10], ref[:10])                  # three pages of 16: the true length
    assert float(got[10:20].float().abs().max()) == 0.0
    assert float(got[20:26].float().abs().max()) == 0.0 and bool((got[26:30].float().abs().amax((1, 2)) > 0).all())


def test_rows_outside_every_sequence_stay(H):
    b = Batch(torch.bfloat16, [100, 64], [30, 5], 4, 2, 64, 16, seed=10)
    q = torch.cat([b.q, torch.full((9, 4, 64), math.nan, device="cuda", dtype=torch.bfloat16)])
    out = torch.full_like(q, 7.0)
    H.attn_paged(q, b.k, b.v, b.table, b.len_t, b.cu, out=out)
    assert torch.equal(out[:35], b.run(H)) and bool((out[35:] == 7.0).all())
    # offsets that leave the batch are cut off at its last row
    cu = b.cu.clone()
    cu[-1] = 10 ** 6
    H.attn_paged(q[:35].contiguous(), b.k, b.v, b.table, b.len_t, cu, out=out[:35])
    assert bool((out[35:] == 7.0).all())


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_launch_hints_do_not_change_what_is_computed(H, dt):
    b = Batch(TYPES[dt], [3000, 200, 17], [40, 1, 17], 4, 2, 128, 32, seed=11)
    want, tol = b.want()
    for max_q, max_len in [(1, 1), (40, 3000), (17, 100), (58, 10 ** 6), (3, 700)]:
        got = b.run(H, max_q=max_q, max_len=max_len)
        assert bool(((got.double() - want).abs() <= tol).all()), (max_q, max_len)


def test_scale_and_the_same_answer_twice(H):
    b = Batch(torch.bfloat16, [2000, 900], [1, 1], 8, 2, 128, 16, seed=12)
    for scale in (0.3, -0.05, 0.0):
        b.check(H, scale=scale)
    assert torch.equal(b.run(H), b.run(H))


def test_offsets_past_32_bits(H):
    """A cache of 5 GB whose pages in use lie at its end."""
    page, kv, D, P = 64, 8, 128, 40000
    pool = torch.empty(P, page, kv, D, dtype=torch.bfloat16, device="cuda")
    b = Batch(torch.bfloat16, [500], [3], 16, kv, D, page, seed=13)
    n = b.k.shape[0]
    pool[P - n:] = b.k
    want = H.attn_paged(b.q, b.k, b.k, b.table, b.len_t, b.cu)
    table = torch.where(b.table >= 0, b.table + (P - n), b.table)
    assert torch.equal(H.attn_paged(b.q, pool, pool, table, b.len_t, b.cu), want)


def test_attention_in_a_graph_on_another_stream(H):
    """Captured once, replayed while the sequences grow; two graphs of different shapes in turn with eager calls between."""
    page, heads, kv, D = 16, 8, 2, 128
    b = Batch(torch.bfloat16, [1200, 700], [1, 1], heads, kv, D, page, seed=14)
    c = Batch(torch.float16, [900, 77, 5], [20, 3, 5], 2, 2, 256, page, seed=15)
    outs = [torch.zeros_like(b.q), torch.zeros_like(c.q)]
    graphs, s = [], torch.cuda.Stream()
    for x, o in zip((b, c), outs):
        x.run(H, out=o)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            x.run(H, out=o)
        graphs.append(g)
    for step in range(4):
        b.lens = [1200 - 100 * step, 700 - 3 * step]
        b.len_t.copy_(torch.tensor(b.lens, dtype=torch.int32))
        wants = [b.run(H), c.run(H)]
        torch.cuda.synchronize()
        for o in outs:
            o.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], wants[0]) and torch.equal(outs[1], wants[1])
        b.rows_k, b.rows_v = [r[:n] for r, n in zip(b.rows_k, b.lens)], [r[:n] for r, n in zip(b.rows_v, b.lens)]
        want, tol = b.want()
        assert bool(((outs[0].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dt", sorted(TYPES))
def test_block_and_window_as_large_as_an_int(H, dt):
    """Blocks longer than any sequence: block is dense, prev sees nothing, transpose sees the query's own position."""
    big = 2 ** 31 - 1
    for nq in ([1, 1], [40, 130]):
        b = Batch(TYPES[dt], [90, 130], nq, 4, 2, 64, 16, seed=16)
        for func, bc, window in [(BLOCK, big, 0), (TRANSPOSE, big, 0), (DENSE, 0, big), (TRANSPOSE, big - 100, 0), (BLOCK, 2 ** 33, 0)]:
            b.check(H, func, bc, window)
        assert float(b.run(H, func=PREV, block_ctx=big).float().abs().max()) == 0.0


@pytest.mark.parametrize("dt", sorted(TYPES))
@pytest.mark.parametrize("page", [5000, 4096, 65536])
def test_one_page_holds_a_whole_sequence(H, dt, page):
    for nq in ([1, 1], [70, 5]):
        Batch(TYPES[dt], [3000, 41], nq, 2, 1, 64, page, seed=17, spare=0).check(H)


def test_two_streams_at_once(H):
    """Calls whose keys are split (each with a workspace of its own) on two streams, neither waiting for the other."""
    a = Batch(torch.bfloat16, [4000, 900], [1, 1], 8, 2, 128, 16, seed=18)
    c = Batch(torch.float16, [2500, 700], [60, 33], 4, 1, 64, 16, seed=19)
    want = [a.run(H), c.run(H)]
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for stream, x, o in ((s, a, outs[0]), (t, c, outs[1])):
            with torch.cuda.stream(stream):
                o.append(x.run(H))
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(w, x) for x in o)


def test_more_sequences_and_heads_than_one_launch_dimension(H):
    """70000 sequences of a few tokens, whose workgroups are more than 65535; the last and the first are right."""
    n, page = 70000, 4
    g = torch.Generator("cuda").manual_seed(20)
    k, v = (torch.randn(n, page, 1, 8, generator=g, device="cuda") for _ in range(2))
    q = torch.randn(n, 2, 8, generator=g, device="cuda")
    table = torch.arange(n, dtype=torch.int32, device="cuda").flip(0)[:, None].contiguous()
    lens = torch.full((n,), 3, dtype=torch.int32, device="cuda")
    got = H.attn_paged(q, k, v, table, lens, torch.arange(n + 1, dtype=torch.int32, device="cuda"), max_q=1)
    kk, vv = (x.flip(0)[:, :3, 0].double() for x in (k, v))
    s = (q.double()[:, :, None] * kk[:, None]).sum(-1) / math.sqrt(8)
    want = (torch.softmax(s, 2)[..., None] * vv[:, None]).sum(2)
    # scores of at most 8 products each (below 20 in all) to 8 2^-24 of theirs, the values' sum to 64 2^-24 of the largest (below 6)
    assert float((got.double() - want).abs().max()) <= (2 * 8 * 20 + 64) * 2.0 ** -24 * 6


def test_a_batch_padded_far_beyond_its_rows(H):
    """A buffer of 300000 rows of which five are queries: split as far as a workspace of 1 GiB allows."""
    b = Batch(torch.bfloat16, [6000, 900], [3, 2], 8, 2, 64, 16, seed=21)
    q = torch.full((300000, 8, 64), math.nan, device="cuda", dtype=torch.bfloat16)
    q[:5] = b.q
    out = torch.full_like(q, 7.0)
    H.attn_paged(q, b.k, b.v, b.table, b.len_t, b.cu, max_q=3, out=out)
    want, tol = b.want()
    assert bool(((out[:5].double() - want).abs() <= tol).all()) and bool((out[5:] == 7.0).all())
