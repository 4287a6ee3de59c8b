"""GPU suite: the paged attention where its inputs are at their limits -- probabilities far below the largest, infinite keys and values that
are seen, table entries that name no page inside a chunk, sizes at the end of what a call may have -- against 64 bits.

The tolerance is test_hip_paged.py's, with the probabilities' own term by the kernel that the call takes:
    |got - want| <= u |want| + (2 ds + dp + n 2^-24) sum_k p_k |v_k| + 2^-39 sum_k |v_k| (half) + half a step of the smallest half
  dp  2^-16 (bfloat16), 2^-22 (half) where the probabilities enter in two parts; 2^-8, 2^-11 in the kernel of chunks (heads of up to 256
      channels, not the transpose pattern, 64 rows and more: max_q * heads / kv); plus 2^-22 for the exponential
  2^-39  halfs below 2^-14 have an absolute step of 2^-24: half of it, of probabilities that enter 2^14 times as large
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_hip_paged import DENSE, TRANSPOSE, TYPES, Batch, visible  # noqa: E402


@pytest.fixture(scope="module")
def H():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from jukebox_amd import _lib, hip_ops
    _lib.lib()          # fail loudly if the extension is missing
    return hip_ops


class Made(Batch):
    """A batch whose rows are given: keys(i), values(i) of sequence i as (len, kv, D), queries as (rows, heads, D)."""

    def __init__(self, dtype, lens, nq, heads, kv, D, page, keys=None, values=None, queries=None, **kw):
        super().__init__(dtype, lens, nq, heads, kv, D, page, **kw)
        for i, n in enumerate(lens):
            pos = torch.arange(n, device="cuda")
            pg = self.table[i, pos // page].long()
            for made, pool, rows in ((keys, self.k, self.rows_k), (values, self.v, self.rows_v)):
                if made is not None:
                    x = made(i).to(dtype)
                    pool[pg, pos % page] = x
                    rows[i] = x.double()
        if queries is not None:
            self.q = queries.to(dtype)

    def chunks(self, func, max_q=None):
        """Whether the call takes the kernel of chunks."""
        if max_q is None:
            max_q = 1 if sum(self.nq) == len(self.nq) else sum(self.nq)
        rows = max_q * self.heads // self.kv
        return self.dtype != torch.float32 and func != TRANSPOSE and self.D <= 256 and rows >= 64

    def fine(self, func=DENSE, bc=0, window=0, max_q=None):
        """(values, tolerances) in 64 bits."""
        scale, u, at = 1.0 / math.sqrt(self.D), torch.finfo(self.dtype).eps / 2, 0
        half, two = self.dtype == torch.float16, not Made.chunks(self, func, max_q)
        dp = {torch.float32: 0.0, torch.float16: 2.0 ** (-22 if two else -11), torch.bfloat16: 2.0 ** (-16 if two else -8)}[self.dtype] + 2.0 ** -22
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        tol = torch.full_like(out, 1e-30)
        for i, (n, nq) in enumerate(zip(self.lens, self.nq)):
            q = self.q[at:at + nq].double()
            see = visible(func, bc, window, torch.arange(n - nq, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None, :])
            for h in range(self.heads):
                k, v = (r[i][:, h * self.kv // self.heads] for r in (self.rows_k, self.rows_v))
                s = torch.where(see, (q[:, h] @ k.T) * scale, -math.inf)
                ds = self.D * 2.0 ** -24 * (q[:, h].abs() @ k.abs().T) * scale + 3 * 2.0 ** -24 * torch.where(see, s.abs(), 0.0)
                p = torch.softmax(s, 1)
                o = p @ v
                # a score's error moves its own probability, and all of them through the sum
                mean = (p * ds).sum(1, keepdim=True)
                out[at:at + nq, h] = o
                tol[at:at + nq, h] += (u * o.abs() + (1 + u) * ((p * ds) @ v.abs() + (mean + dp + (n / 64 + 64) * 2.0 ** -24) * (p @ v.abs()))
                                       + (2.0 ** -39 * (see.double() @ v.abs()) + 2.0 ** -25 if half else 0.0))
            at += nq
        return out, tol

    def check_fine(self, H, **kw):
        got = self.run(H, **{{"bc": "block_ctx"}.get(k, k): v for k, v in kw.items()})
        torch.cuda.synchronize()
        want, tol = self.fine(**kw)
        off = (got.double() - want).abs()
        assert bool((off <= tol).all()), f"off by {float((off / tol).max()):.3g} tolerances, {int((~(off <= tol)).sum())} of {off.numel()} elements"


@pytest.mark.parametrize("dt", sorted(TYPES))
@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("heads,kv,D,lens,nq,kw", [
    (2, 2, 64, [5, 7], [1, 1], {}), (4, 2, 128, [6], [2], {}), (1, 1, 250, [5], [3], {}), (1, 1, 480, [7], [2], {}), (3, 3, 300, [40], [34], {"window": 5}),
    (2, 1, 40, [90], [80], {"func": TRANSPOSE, "bc": 20}), (1, 1, 480, [100], [90], {"window": 6}), (2, 1, 64, [100], [70], {"window": 5})],
    ids=["one", "two", "250", "480", "300", "transpose", "chunk480", "chunk64"])
def test_values_that_cancel(H, dt, page, heads, kv, D, lens, nq, kw):
    """Neighbouring values of opposite signs, so that an output is far below what its products add up to and the probabilities' own
    rounding shows.  Few keys a query, short queries: the scores' error is below it."""
    g = torch.Generator("cuda").manual_seed(D)

    def values(i):
        n = lens[i]
        sign = 1.0 - 2.0 * (torch.arange(n, device="cuda") // (20 if kw.get("func") == TRANSPOSE else 1) % 2)
        return sign[:, None, None] * (1 + 0.01 * torch.randn(n, kv, D, generator=g, device="cuda"))

    q = 0.5 / math.sqrt(D) * torch.randn(sum(nq), heads, D, generator=g, device="cuda")
    Made(TYPES[dt], lens, nq, heads, kv, D, page, values=values, queries=q, seed=D).check_fine(H, **kw)


def peaked(dt, heads, kv, D, lens, nq, page, nats, seed):
    """The first key of every sequence `nats` above thousands of others; its value 0, the others' 1."""
    g = torch.Generator("cuda").manual_seed(seed)

    def keys(i):
        k = 0.01 * torch.randn(lens[i], kv, D, generator=g, device="cuda")
        k[:, :, 0] = -nats
        k[0, :, 0] = 0.0
        return k

    def values(i):
        v = torch.ones(lens[i], kv, D, device="cuda")
        v[0] = 0.0
        return v

    q = 0.1 * torch.randn(sum(nq), heads, D, generator=g, device="cuda")
    q[:, :, 0] = math.sqrt(D)
    return Made(TYPES[dt], lens, nq, heads, kv, D, page, keys=keys, values=values, queries=q, seed=seed)


@pytest.mark.parametrize("dt", sorted(TYPES))
@pytest.mark.parametrize("nats", [8.0, 14.0, 17.0, 17.5, 18.0, 20.0, 24.0])
@pytest.mark.parametrize("heads,kv,D,lens,nq,page", [
    (2, 2, 64, [8000], [1], 16), (2, 1, 128, [5000, 3001], [2, 1], 7), (1, 1, 480, [4096], [1], 64), (1, 1, 256, [4096, 77], [3, 1], 16),
    (1, 1, 64, [8000], [80], 16), (4, 2, 128, [3000, 600], [200, 40], 20), (2, 2, 150, [2500], [130], 32), (1, 1, 256, [3000], [70], 16), (8, 8, 64, [2000] * 40, [1] * 40, 16)],
    ids=["one", "few", "480", "256", "chunk64", "chunk128", "chunk150", "chunk256", "batch"])
def test_one_key_far_above_thousands(H, dt, nats, heads, kv, D, lens, nq, page):
    """An attention sink: the long tail's share, far below 2^-14, carries the whole output."""
    peaked(dt, heads, kv, D, lens, nq, page, nats, seed=D).check_fine(H)


@pytest.mark.parametrize("dt", sorted(TYPES))
@pytest.mark.parametrize("nq", [1, 80])
@pytest.mark.parametrize("size", [40.0, 1000.0])
def test_scores_far_from_zero(H, dt, nq, size):
    """Scores of 10^4 and 10^7, up and down: one key takes all, the others nothing, and no probability passes the type's range."""
    for D in (64, 480):
        for sign in (1.0, -1.0):
            n = 200
            step = torch.arange(n, device="cuda").double() / n

            def keys(i):
                k = torch.zeros(n, 1, D, device="cuda")
                k[:, 0, :] = (sign * size * (1 + step))[:, None]
                return k

            b = Made(TYPES[dt], [n], [nq], 1, 1, D, 16, keys=keys, queries=torch.full((nq, 1, D), size, device="cuda"), seed=5)
            got = b.run(H).double()
            s = (b.q[:, 0].double() @ b.rows_k[0][:, 0].T) / math.sqrt(D)
            for r in range(nq):
                seen = n - nq + r + 1
                # (rows of one rounded value tie exactly; they share)
                p = torch.softmax(s[r, :seen], 0)
                want = p @ b.rows_v[0][:seen, 0]
                assert float((got[r, 0] - want).abs().max()) <= 2.0 ** -7 * 6, (size, sign, r)


@pytest.mark.parametrize("dt", sorted(TYPES))
@pytest.mark.parametrize("nq", [1, 80])
@pytest.mark.parametrize("page", [16, 7])
def test_scores_past_what_a_float_tells_apart(H, dt, nq, page):
    """Scores of 10^9 .. 10^12, whose fused product and the rounded one they are taken from are hundreds apart: still an average of values,
    that of the largest score where it stands clear of the others."""
    for D in (64, 480):
        for sign in (1.0, -1.0):
            for size in (10000.0, 60000.0) + ((1e6,) if dt != "f16" else ()):
                n, top = 150, 40

                def keys(i):
                    k = torch.full((n, 1, D), -sign * size, device="cuda")
                    k[top] = sign * size if sign > 0 else -0.5 * sign * size
                    return k

                q = torch.full((nq, 1, D), size, device="cuda")
                q[..., ::3] *= 0.77
                b = Made(TYPES[dt], [n], [nq], 1, 1, D, page, keys=keys, queries=q, seed=6)
                got = b.run(H).double()
                s = (b.q[:, 0].double() @ b.rows_k[0][:, 0].T)
                for r in range(nq):
                    seen = n - nq + r + 1
                    tie = s[r, :seen] == s[r, :seen].max()          # one key, or all the others: equal rows
                    want = b.rows_v[0][:seen, 0][tie].mean(0)
                    assert float((got[r, 0] - want).abs().max()) <= 2.0 ** -7 * 6, (D, sign, size, r)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,D", [(2, 2, 64), (4, 2, 128), (2, 2, 150), (1, 1, 256), (2, 1, 40), (1, 1, 200)])
@pytest.mark.parametrize("page", [16, 10, 64])
def test_missing_pages_in_chunks(H, dt, heads, kv, D, page):
    """Table entries that name no page, in turns that every row sees and in the diagonal ones; then with NaN and infinity in rows of pages
    that are there, beside the missing ones: they reach the queries that see them, and no others."""
    n, nq = 500, 170
    b = Batch(TYPES[dt], [n, 90], [nq, 90], heads, kv, D, page, seed=D + page)
    table, gone = b.table.clone(), (100 // page, (n - 60) // page)
    table[0, gone[0]], table[0, gone[1]], table[1, 30 // page] = -1, 10 ** 6, b.k.shape[0]
    b.table = table

    def blind(i, pos):
        p = pos // page
        return (p == gone[0]) | (p == gone[1]) if i == 0 else p == 30 // page

    got = b.run(H)
    want, tol = b.want(blind=blind)
    assert bool(((got.double() - want).abs() <= tol).all())
    # a value beside the first gap (seen by all rows), one beside the second (by the last ones)
    beside = [gone[0] * page - 1, (gone[1] + 1) * page]
    for what in (math.nan, math.inf):
        for pos in beside:
            pg, keep = int(table[0, pos // page]), b.v[int(table[0, pos // page]), pos % page].clone()
            b.v[pg, pos % page, :, D // 3] = what
            odd = b.run(H)
            b.v[pg, pos % page] = keep
            sees = torch.arange(n - nq, n, device="cuda") >= pos
            hit = odd[:nq, :, D // 3].float()
            assert bool((~torch.isfinite(hit[sees])).all()), (what, pos)
            clean = torch.ones_like(odd, dtype=torch.bool)
            clean[:nq][sees, :, D // 3] = False
            assert bool(((odd.double() - want).abs() <= tol)[clean].all()), (what, pos)


def seen_infinities(b, func, bc):
    """(values, tolerances) in 64 bits, product by product: infinite keys and values as the definition has them."""
    scale, u, at = 1.0 / math.sqrt(b.D), torch.finfo(b.dtype).eps / 2, 0
    dp = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[b.dtype] + 2.0 ** -22
    out = torch.zeros(b.q.shape, dtype=torch.float64, device="cuda")
    tol = torch.full_like(out, 1e-30)
    for i, (n, nq) in enumerate(zip(b.lens, b.nq)):
        q = b.q[at:at + nq].double()
        see = visible(func, bc, 0, torch.arange(n - nq, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None, :])
        for h in range(b.heads):
            k, v = (r[i][:, h * b.kv // b.heads] for r in (b.rows_k, b.rows_v))
            fk, fv = (torch.where(torch.isfinite(x), x, 0.0) for x in (k, v))
            for r in range(nq):
                s = torch.where(see[r], (q[r, h] * k).sum(1) * scale, -math.inf)
                ds = b.D * 2.0 ** -24 * (q[r, h].abs() * fk.abs()).sum(1).max() * scale + 3 * 2.0 ** -24 * float(torch.where(torch.isfinite(s), s.abs(), 0.0).max())
                p = torch.softmax(s, 0)
                out[at + r, h] = torch.where(see[r][:, None] & (p != 0)[:, None], p[:, None] * v, 0.0).sum(0)
                whole = torch.where(see[r], p, 0.0)[:, None].nan_to_num() * fv.abs()
                tol[at + r, h] += u * out[at + r, h].abs().nan_to_num(posinf=0.0) + (2 * ds + dp + (n / 64 + 64) * 2.0 ** -24) * whole.sum(0) * (1 + u) + (
                    2.0 ** -24 if b.dtype == torch.float16 else 0.0)
        at += nq
    return out, tol


@pytest.mark.parametrize("dt", sorted(TYPES))
@pytest.mark.parametrize("what", ["value", "values", "key"])
@pytest.mark.parametrize("heads,kv,D,lens,nq,page,func,bc", [
    (2, 2, 64, [100], [1], 16, DENSE, 0), (4, 2, 128, [100, 70], [1, 3], 16, DENSE, 0), (3, 3, 33, [90], [2], 7, DENSE, 0), (1, 1, 150, [200], [1], 16, DENSE, 0),
    (1, 1, 250, [130], [5], 20, DENSE, 0), (1, 1, 480, [150], [1], 64, DENSE, 0), (2, 1, 300, [90], [34], 16, DENSE, 0), (2, 1, 128, [5000], [1], 16, DENSE, 0),
    (2, 2, 64, [300], [70], 16, DENSE, 0), (2, 2, 150, [260], [66], 32, DENSE, 0), (1, 1, 40, [300], [80], 10, DENSE, 0), (4, 2, 250, [200], [40], 16, DENSE, 0),
    (1, 1, 64, [2100], [70], 64, DENSE, 0), (2, 1, 50, [120], [90], 16, TRANSPOSE, 20)],
    ids=["one64", "one128", "few33", "one150", "few250", "one480", "chunk300", "split", "chunk64", "chunk150", "chunk40", "chunk250", "splitchunk", "transpose"])
def test_infinities_that_are_seen(H, dt, what, heads, kv, D, lens, nq, page, func, bc):
    """An infinite value in an output's sum makes it infinite (two of both signs: no number); an infinite channel of a key makes its score
    infinite: -inf takes the key out, +inf leaves no number.  Whatever the turn, the kernel, and the channel, a head's last ones too."""
    for where in (D - 1, D - 8, D // 2, 0):
        b = Batch(TYPES[dt], lens, nq, heads, kv, D, page, seed=D + where)
        for pos, sign in [(5, -1.0)] + ([(8, 1.0)] if what == "values" else []):
            pos = pos if func == DENSE else pos * bc // 5        # (the transpose pattern: positions of one residue)
            x, rows = (b.k, b.rows_k) if what == "key" else (b.v, b.rows_v)
            x[int(b.table[0, pos // page]), pos % page, :, where] = sign * math.inf
            rows[0][pos, :, where] = sign * math.inf
        got = b.run(H, func=func, block_ctx=bc).double()
        want, tol = seen_infinities(b, func, bc)
        nan, inf = torch.isnan(want), torch.isinf(want)
        assert bool(torch.isnan(got).eq(nan).all()), f"{int((torch.isnan(got) != nan).sum())} of {nan.numel()} are (no) numbers, channel {where}"
        assert torch.equal(got[inf], want[inf])
        fine = ~nan & ~inf
        assert bool(((got - want).abs() <= tol)[fine].all()), where
        assert what != "value" or bool(inf.any())


@pytest.mark.parametrize("dt", sorted(TYPES))
@pytest.mark.parametrize("nats", [30.0, 75.0])
@pytest.mark.parametrize("heads,kv,D,lens,nq,page", [(2, 2, 64, [300], [1], 16), (2, 1, 128, [6000], [1], 16), (1, 1, 480, [200], [3], 7), (1, 1, 150, [300], [80], 16), (1, 1, 64, [2100], [70], 16)],
                         ids=["one", "split", "480", "chunk", "splitchunk"])
def test_an_infinite_value_of_a_probability_that_is_nearly_none(H, dt, nats, heads, kv, D, lens, nq, page):
    """e^-30 and e^-75 of an infinite value are infinite, in whatever part of the keys it lies."""
    for pos in (5, lens[0] - 90):
        b = peaked(dt, heads, kv, D, lens, nq, page, nats, seed=D)
        want, tol = b.fine()
        b.v[int(b.table[0, pos // page]), pos % page, :, D - 3] = -math.inf
        got = b.run(H).double()
        assert bool((got[:, :, D - 3] == -math.inf).all()), pos
        rest = torch.arange(D, device="cuda") != D - 3
        assert bool(((got - want).abs() <= tol)[..., rest].all()), pos


@pytest.mark.parametrize("page", [2 ** 30 + 1, 2 ** 30 + 16, 2 ** 31 - 1])
def test_one_page_of_more_than_2_30_rows(H, page):
    """A page of more rows than 2^30, all of them the same one in memory (a row stride of 0): the average is the row."""
    for dt, D, nq in (("f16", 8, 1), ("bf16", 64, 70), ("f32", 16, 2)):
        row = torch.randn(2, 1, 1, 1, D, device="cuda").to(TYPES[dt])
        k, v = (x.expand(1, page, 1, D) for x in row)
        q = torch.randn(nq, 1, D, device="cuda").to(TYPES[dt])
        ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        got = H.attn_paged(q, k, v, ints([0]), ints(5000), ints(0, nq), max_len=5000)
        # probabilities that sum to 1 but for their own rounding and that of 5000 / 64 + 64 additions
        dp = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dt]
        u = torch.finfo(TYPES[dt]).eps / 2
        assert float(((got.double() - v[0, 0].double()).abs() / v[0, 0].double().abs()).max()) <= u + (1 + u) * (dp + (5000 / 64 + 64) * 2.0 ** -24)


@pytest.mark.parametrize("dt", sorted(TYPES))
def test_hints_of_zero(H, dt):
    """max_q and max_len below the truth cost time, not correctness: 0 too."""
    b = Batch(TYPES[dt], [300, 17], [5, 17], 4, 2, 64, 16, seed=31)
    want, tol = b.want()
    for kw in ({"max_q": 0}, {"max_len": 0}, {"max_q": 0, "max_len": 0}):
        got = H.attn_paged(b.q, b.k, b.v, b.table, b.len_t, b.cu, out=torch.full_like(b.q, 7.0), **kw)
        assert bool(((got.double() - want).abs() <= tol).all()), kw


@pytest.mark.parametrize("dt", sorted(TYPES))
def test_hints_far_beyond_the_truth(H, dt):
    """70000 sequences of one token, and max_q for as many: more tiles than a launch holds workgroups."""
    n, page = 70000, 4
    g = torch.Generator("cuda").manual_seed(20)
    k, v = (torch.randn(n, page, 1, 8, generator=g, device="cuda").to(TYPES[dt]) for _ in range(2))
    q = torch.randn(n, 2, 8, generator=g, device="cuda").to(TYPES[dt])
    table = torch.arange(n, dtype=torch.int32, device="cuda").flip(0)[:, None].contiguous()
    lens = torch.full((n,), 3, dtype=torch.int32, device="cuda")
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    want = H.attn_paged(q, k, v, table, lens, cu, max_q=1)
    got = H.attn_paged(q, k, v, table, lens, cu, max_q=n)
    # three values below 6, with probabilities off by their rounding in either call
    u = torch.finfo(TYPES[dt]).eps / 2
    assert float((got.double() - want.double()).abs().max()) <= (4 * u + 2.0 ** -18) * 6
    # one sequence has the queries of all, in turns of the tiles that are left
    cu[1:] = n
    lens[0] = 3
    first = H.attn_paged(q, k, v, table, lens, cu, max_q=n)
    assert bool((first[:-3] == 0).all()) and bool((first[-3:].abs().sum((1, 2)) > 0).all())


def test_a_step_without_max_q(H):
    """One token of each of many sequences: without max_q the call is the one of few tokens (the same bits), not the one of chunks."""
    lens = [700, 33, 5, 1200] * 16
    for heads, kv, D in ((8, 2, 128), (2, 2, 64), (16, 1, 64)):
        b = Batch(torch.bfloat16, lens, [1] * 64, heads, kv, D, 16, seed=40)
        assert torch.equal(b.run(H), b.run(H, max_q=1))
        want, tol = Made.fine(b)
        assert bool(((b.run(H).double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dt", sorted(TYPES))
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-3, 2.0])
@pytest.mark.parametrize("heads,kv,D", [(2, 2, 9), (2, 1, 12), (1, 1, 15), (2, 2, 23), (2, 2, 150), (1, 1, 200), (1, 1, 255), (1, 1, 301)])
def test_scales_and_odd_widths(H, dt, scale, heads, kv, D):
    """Negative, zero and large scales; heads whose last piece repeats 1 to 7 channels, in one piece more than they fill and in many."""
    for lens, nq, page in (([90, 33], [1, 1], 16), ([300, 20], [80, 20], 7), ([700], [100], 64)):
        Batch(TYPES[dt], lens, nq, heads, kv, D, page, seed=D).check(H, scale=scale)


def test_a_table_that_is_part_of_a_wider_one(H):
    b = Batch(torch.bfloat16, [300, 41, 7], [70, 1, 3], 4, 2, 64, 16, seed=50)
    wide = torch.full((3, b.table.shape[1] + 9), 10 ** 6, dtype=torch.int32, device="cuda")
    wide[:, 4:4 + b.table.shape[1]] = b.table
    want = b.run(H)
    b.table = wide[:, 4:4 + b.table.shape[1]]
    assert torch.equal(b.run(H), want)
