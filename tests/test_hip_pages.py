"""GPU suite: rows into pages and the control of the pages, against a model of it in plain Python; every number has to be equal."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

NONE_FREE, BAD_ARG = 1, 2


@pytest.fixture(scope="module")
def H():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from jukebox_amd import _lib, hip_ops
    _lib.lib()          # fail loudly if the extension is missing
    return hip_ops


def ints(v, kind=torch.int32):
    return torch.tensor(v, dtype=kind, device="cuda")


class Model:
    """What the calls do, one page and one row at a time."""

    def __init__(self, n_seq, max_pages, n_pages, page, pools):
        self.table = [[-1] * max_pages for _ in range(n_seq)]
        self.lens, self.ref, self.page, self.max_pages, self.status = [0] * n_seq, [0] * n_pages, page, max_pages, 0
        self.pools = [p.cpu().clone() for p in pools]

    def free_pages(self):
        return [p for p, c in enumerate(self.ref) if c == 0]

    def pages(self, n):
        return -(-n // self.page)

    def extend(self, news, n_tokens):
        need = [self.pages(n + m) - self.pages(n) for n, m in zip(self.lens, news)]
        if any(self.pages(n + m) > self.max_pages for n, m in zip(self.lens, news)):
            self.status = BAD_ARG
            return [-1] * n_tokens
        free = self.free_pages()
        if sum(need) > len(free):
            self.status = NONE_FREE
            return [-1] * n_tokens
        slots = []
        for i, m in enumerate(news):
            for t in range(m):
                pos = self.lens[i] + t
                if pos % self.page == 0:
                    p = free.pop(0)
                    self.table[i][pos // self.page], self.ref[p] = p, 1
                slots.append(self.table[i][pos // self.page] * self.page + pos % self.page)
            self.lens[i] += m
        return slots + [-1] * (n_tokens - len(slots))

    def free(self, rows):
        if len(set(rows)) != len(rows) or any(not 0 <= r < len(self.lens) for r in rows):
            self.status = BAD_ARG
            return
        for r in rows:
            for p in self.table[r]:
                if p >= 0:
                    self.ref[p] -= 1
            self.table[r], self.lens[r] = [-1] * self.max_pages, 0

    def fork(self, src, dst):
        rows = range(len(self.lens))
        if (len(set(dst)) != len(dst) or any(r not in rows for r in src + dst) or set(src) & set(dst) or any(self.lens[d] for d in dst)):
            self.status = BAD_ARG
            return
        free = self.free_pages()
        if sum(self.lens[s] % self.page > 0 for s in src) > len(free):
            self.status = NONE_FREE
            return
        for s, d in zip(src, dst):
            n = self.lens[s]
            for c in range(self.pages(n)):
                p = self.table[s][c]
                if (c + 1) * self.page > n:
                    q = free.pop(0)
                    for x in self.pools:
                        x[q] = x[p]
                    p = q
                self.table[d][c] = p
                self.ref[p] += 1
            self.lens[d] = n

    def compact(self):
        live = sum(c > 0 for c in self.ref)
        holes = [p for p in range(live) if self.ref[p] == 0]
        to = {}
        for p in range(live, len(self.ref)):
            if self.ref[p] > 0:
                q = to[p] = holes.pop(0)
                self.ref[q], self.ref[p] = self.ref[p], 0
                for x in self.pools:
                    x[q] = x[p]
        self.table = [[to.get(p, p) for p in r] for r in self.table]


class Device:
    def __init__(self, H, n_seq, max_pages, n_pages, page, pools):
        self.H, self.pools, self.page = H, pools, page
        self.table, self.lens, self.ref = ints([[-1] * max_pages] * n_seq), ints([0] * n_seq), ints([0] * n_pages)
        self.status = ints([0])

    def same(self, m):
        torch.cuda.synchronize()
        assert int(self.status) == m.status
        assert self.lens.tolist() == m.lens
        assert self.table.tolist() == m.table
        assert self.ref.tolist() == m.ref
        for x, y in zip(self.pools, m.pools):
            assert torch.equal(x.cpu(), y)


def make(H, n_seq, max_pages, n_pages, page, width=24, n_pools=2, dtype=torch.float16):
    g = torch.Generator("cuda").manual_seed(n_pages)
    pools = [torch.randn(n_pages, page, width, generator=g, device="cuda").to(dtype) for _ in range(n_pools)]
    return Device(H, n_seq, max_pages, n_pages, page, pools), Model(n_seq, max_pages, n_pages, page, pools)


@pytest.mark.parametrize("n_seq,max_pages,n_pages,page,seed", [(5, 6, 20, 4, 0), (40, 9, 150, 16, 1), (3, 40, 64, 1, 2), (1, 3, 2, 7, 3), (1500, 4, 5000, 5, 4)])
def test_a_run_of_calls_follows_the_model(H, n_seq, max_pages, n_pages, page, seed):
    """Extend, fork, free and compact in random order, running out of pages and refusing now and then."""
    rng = np.random.default_rng(seed)
    d, m = make(H, n_seq, max_pages, n_pages, page)
    for step in range(40 if n_seq < 1000 else 8):
        what = rng.integers(0, 8)
        if what < 4:
            news = [int(rng.integers(0, 2 * page + 1)) if rng.random() < 0.6 else 0 for _ in range(n_seq)]
            extra = int(rng.integers(0, 5))
            cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
            slots = H.pages_extend(d.table, d.lens, d.ref, ints(cu.tolist()), page, int(cu[-1]) + extra, d.status)
            assert slots.tolist() == m.extend(news, int(cu[-1]) + extra)
        elif what < 6:
            k = int(rng.integers(0, n_seq + 1))
            rows = rng.permutation(n_seq)[:k].tolist()
            H.pages_free(d.table, d.lens, d.ref, ints(rows), d.status)
            m.free(rows)
        elif what == 6:
            order = rng.permutation(n_seq).tolist()
            empty = [r for r in order if m.lens[r] == 0]
            full = [r for r in order if m.lens[r] > 0] or order[:1]
            k = int(rng.integers(0, len(empty) + 1))
            dst = empty[:k]
            src = [full[int(rng.integers(0, len(full)))] for _ in dst]
            H.pages_fork(d.pools, d.table, d.lens, d.ref, ints(src), ints(dst), page, d.status)
            m.fork(src, dst)
        else:
            d.table, d.ref = H.pages_compact(d.pools, d.table, d.ref)
            m.compact()
        d.same(m)
        d.status.zero_()
        m.status = 0


def test_calls_that_cannot_be_done_change_nothing_but_the_status(H):
    d, m = make(H, 4, 4, 10, 4)
    H.pages_extend(d.table, d.lens, d.ref, ints([0, 7, 9, 9, 9]), 4, 9, d.status)
    m.extend([7, 2, 0, 0], 9)
    d.same(m)
    for cu, code in [([0, 9, 9, 9, 9], 0), ([0, 10, 10, 10, 10], BAD_ARG), ([0, 9, 20, 30, 30], NONE_FREE), ([0, 3, 2, 4, 4], BAD_ARG), ([1, 2, 2, 2, 2], BAD_ARG),
                     ([0, 1, 1, 1, 40], BAD_ARG)]:
        if code == 0:
            continue
        slots = H.pages_extend(d.table, d.lens, d.ref, ints(cu), 4, 30, d.status)
        assert slots.tolist() == [-1] * 30 and int(d.status) == code
        d.status.zero_()
        d.same(m)
    for rows in ([0, 0], [4], [-1, 1]):
        H.pages_free(d.table, d.lens, d.ref, ints(rows), d.status)
        assert int(d.status) == BAD_ARG
        d.status.zero_()
        d.same(m)
    for src, dst in [([0], [1]), ([0, 0], [2, 2]), ([0], [4]), ([9], [2]), ([2, 0], [3, 2])]:
        H.pages_fork(d.pools, d.table, d.lens, d.ref, ints(src), ints(dst), 4, d.status)
        assert int(d.status) == BAD_ARG
        d.status.zero_()
        d.same(m)
    # no page left for the copy of the part-filled one
    H.pages_extend(d.table, d.lens, d.ref, ints([0, 0, 14, 26, 26]), 4, 26, d.status)
    m.extend([0, 14, 12, 0], 26)
    d.same(m)
    H.pages_free(d.table, d.lens, d.ref, ints([3]), d.status)
    H.pages_extend(d.table, d.lens, d.ref, ints([0, 9, 9, 9, 9]), 4, 9, d.status)
    m.free([3])
    m.extend([9, 0, 0, 0], 9)
    d.same(m)


def test_a_length_that_does_not_fit_its_row_is_refused(H):
    d, m = make(H, 3, 2, 10, 4)
    d.lens[1] = 100
    H.pages_fork(d.pools, d.table, d.lens, d.ref, ints([1]), ints([2]), 4, d.status)
    assert int(d.status) == BAD_ARG
    d.lens[1] = -3
    slots = H.pages_extend(d.table, d.lens, d.ref, ints([0, 1, 2, 3]), 4, 3, d.status)
    assert slots.tolist() == [-1] * 3 and int(d.status) == BAD_ARG and d.table.max() == -1


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("KV,D,page,layout", [(8, 128, 16, "nhd"), (2, 256, 64, "hnd"), (1, 480, 20, "nhd"), (8, 150, 1, "nhd"), (5, 33, 7, "hnd"), (1, 8, 3, "nhd"), (40, 4, 5, "nhd")])
def test_write(H, dt, KV, D, page, layout):
    P, T = 50, 37
    g = torch.Generator("cuda").manual_seed(D)
    shape = (2, P, KV, page, D) if layout == "hnd" else (2, P, page, KV, D)
    store = torch.randn(shape, generator=g, device="cuda").to(dt)
    kp, vp = [x.transpose(1, 2) if layout == "hnd" else x for x in store]
    qkv = torch.randn(T, 3, KV, D, generator=g, device="cuda").to(dt)            # rows of one projection's output
    k, v = qkv[:, 1], qkv[:, 2]
    slots = torch.randperm(P * page, generator=torch.Generator().manual_seed(3))[:T].cuda() if P * page >= T else None
    slots = slots.long()
    slots[3], slots[T - 1] = -1, P * page + 5
    want_k, want_v = kp.clone(), vp.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < P * page:
            want_k[s // page, s % page], want_v[s // page, s % page] = k[t], v[t]
    H.kv_write(k, v, kp, vp, slots)
    torch.cuda.synchronize()
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)
    H.kv_write(k[:0], v[:0], kp, vp, slots[:0])


def test_write_past_32_bits(H):
    P, page, KV, D = 40000, 64, 8, 128
    pool = torch.zeros(P, page, KV, D, dtype=torch.bfloat16, device="cuda")
    k = torch.randn(3, KV, D, device="cuda").bfloat16()
    slots = ints([P * page - 1, P * page - 65, 0], torch.int64)
    H.kv_write(k, k, pool, pool, slots)
    assert torch.equal(pool[-1, -1], k[0]) and torch.equal(pool[-2, -1], k[1]) and torch.equal(pool[0, 0], k[2])
    H.pages_copy([pool], ints([P - 1]), ints([P - 3]))
    assert torch.equal(pool[P - 3], pool[P - 1]) and float(pool[P - 4].abs().max()) == 0.0


@pytest.mark.parametrize("dt,shape", [(torch.float16, (30, 16, 480)), (torch.float32, (9, 3, 5)), (torch.uint8, (20, 7)), (torch.uint8, (11, 33, 3)), (torch.bfloat16, (40, 10, 1200))])
@pytest.mark.parametrize("n_pools", [1, 3, 300])
def test_copy(H, dt, shape, n_pools):
    g = torch.Generator("cuda").manual_seed(n_pools)
    store = torch.randint(0, 200, (n_pools, shape[0], 2) + shape[1:], generator=g, device="cuda").to(dt)
    pools = [x[:, 0] for x in store]                                             # every second page is another's
    want = store.clone()
    src, dst = [0, 5, 5, shape[0], 2, -1], [1, 3, 4, 6, shape[0] + 7, 7]
    for a, b in zip(src, dst):
        if 0 <= a < shape[0] and 0 <= b < shape[0]:
            want[:, b, 0] = want[:, a, 0]
    H.pages_copy(pools, ints(src), ints(dst))
    torch.cuda.synchronize()
    assert torch.equal(store, want)
    H.pages_copy(pools, ints([]), ints([]))


def test_more_pools_than_one_launch_takes(H):
    d, m = make(H, 3, 5, 12, 4, width=9, n_pools=300)
    H.pages_extend(d.table, d.lens, d.ref, ints([0, 6, 17, 17]), 4, 17, d.status)
    m.extend([6, 11, 0], 17)
    H.pages_fork(d.pools, d.table, d.lens, d.ref, ints([1]), ints([2]), 4, d.status)
    m.fork([1], [2])
    d.same(m)
    H.pages_free(d.table, d.lens, d.ref, ints([0]), d.status)
    m.free([0])
    d.table, d.ref = H.pages_compact(d.pools, d.table, d.ref)
    m.compact()
    d.same(m)


def test_extend_of_many_tokens_and_scattered_free_pages(H):
    """More tokens than the planning workgroup handles by itself, free pages far apart."""
    n_seq, page, n_pages = 7, 16, 9000
    d, m = make(H, n_seq, 400, n_pages, page, width=1, n_pools=1)
    rng = np.random.default_rng(0)
    taken = rng.random(n_pages) < 0.9
    d.ref.copy_(ints(taken.astype(np.int32).tolist()))
    m.ref = taken.astype(int).tolist()
    for news in ([3000, 0, 1, 16, 17, 4000, 5], [1, 2, 3, 4, 5, 6, 7]):
        cu = np.concatenate([[0], np.cumsum(news)]).tolist()
        slots = H.pages_extend(d.table, d.lens, d.ref, ints(cu), page, cu[-1], d.status)
        assert slots.tolist() == m.extend(news, cu[-1])
        d.same(m)


def test_serving_run_equals_full_attention(H):
    """The calls as they are used together: prompts admitted, written and attended to, tokens added one by one, some sequences forked
    and others ended, the pool compacted on the way; a captured step (extend, write, attend) in between.  Every output against
    64-bit attention over the sequence's whole history."""
    import test_hip_paged as A
    KV, heads, D, page, n_pages, n_seq, max_pages = 2, 6, 64, 8, 60, 6, 12
    g = torch.Generator("cuda").manual_seed(0)
    kp, vp = (torch.full((n_pages, page, KV, D), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    table, lens, ref, status = ints([[-1] * max_pages] * n_seq), ints([0] * n_seq), ints([0] * n_pages), ints([0])
    hist = [[torch.zeros(0, KV, D, device="cuda", dtype=torch.bfloat16) for _ in range(2)] for _ in range(n_seq)]
    q1, k1, v1 = (torch.zeros(n_seq, h, D, device="cuda", dtype=torch.bfloat16) for h in (heads, KV, KV))
    cu1, o1 = ints([0] * (n_seq + 1)), torch.zeros(n_seq, heads, D, device="cuda", dtype=torch.bfloat16)

    def step(q, k, v, cu, out=None):
        slots = H.pages_extend(table, lens, ref, cu, page, q.shape[0], status)
        H.kv_write(k, v, kp, vp, slots)
        return H.attn_paged(q, kp, vp, table, lens, cu, out=out)

    def check(out, q, news):
        at = 0
        for i, m in enumerate(news):
            if m:
                b = A.Batch.__new__(A.Batch)
                n = hist[i][0].shape[0]
                b.dtype, b.lens, b.nq, b.D, b.kv, b.heads = torch.bfloat16, [n], [m], D, KV, heads
                b.q, b.rows_k, b.rows_v = q[at:at + m], [hist[i][0].double()], [hist[i][1].double()]
                want, tol = b.want()
                assert bool(((out[at:at + m].double() - want).abs() <= tol).all())
            at += m
        assert int(status) == 0

    def admit(news):
        T = sum(news)
        q, k, v = (torch.randn(T, h, D, generator=g, device="cuda").bfloat16() for h in (heads, KV, KV))
        cu = np.concatenate([[0], np.cumsum(news)]).tolist()
        for i in range(n_seq):
            hist[i] = [torch.cat([h, x[cu[i]:cu[i + 1]]]) for h, x in zip(hist[i], (k, v))]
        check(step(q, k, v, ints(cu)), q, news)

    admit([17, 8, 0, 3, 0, 30])
    # the captured step: buffers of n_seq tokens, whose number a replay takes from cu1
    step(q1, k1, v1, cu1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(q1, k1, v1, cu1, out=o1)

    def replay(active):
        T = len(active)
        for buf in (q1, k1, v1):
            buf.copy_(torch.randn(buf.shape, generator=g, device="cuda"))
        news = [1 if i in active else 0 for i in range(n_seq)]
        cu1.copy_(ints(np.concatenate([[0], np.cumsum(news)]).tolist()))
        for t, i in enumerate(sorted(active)):
            hist[i] = [torch.cat([h, x[t:t + 1]]) for h, x in zip(hist[i], (k1, v1))]
        graph.replay()
        torch.cuda.synchronize()
        check(o1[:T], q1[:T], news)

    for _ in range(5):
        replay({0, 1, 3, 5})
    H.pages_fork([kp, vp], table, lens, ref, ints([0, 5]), ints([2, 4]), page, status)
    hist[2], hist[4] = list(hist[0]), list(hist[5])
    for _ in range(4):
        replay({0, 2, 4, 5})
    admit([0, 1, 9, 0, 1, 0])
    H.pages_free(table, lens, ref, ints([0, 3]), status)
    hist[0], hist[3] = ([x[:0] for x in h] for h in (hist[0], hist[3]))
    t2, r2 = H.pages_compact([kp, vp], table, ref)
    table.copy_(t2)
    ref.copy_(r2)
    live = int((ref > 0).sum())
    assert bool((ref[:live] > 0).all())
    for _ in range(9):
        replay({1, 2, 4, 5})
    admit([20, 0, 0, 5, 0, 0])
    H.pages_free(table, lens, ref, ints([0, 1, 2, 3, 4, 5]), status)
    assert int(ref.abs().max()) == 0 and int(table.max()) == -1 and int(lens.max()) == 0


def test_calls_with_nothing_to_do(H):
    d, _ = make(H, 3, 4, 10, 16)
    before = [x.clone() for x in (d.table, d.lens, d.ref)]
    assert H.pages_extend(d.table, d.lens, d.ref, ints([0, 0, 0, 0]), 16, 0, d.status).numel() == 0
    assert H.pages_extend(d.table, d.lens, d.ref, ints([0, 0, 0, 0]), 16, 5, d.status).tolist() == [-1] * 5
    none = ints([])
    H.pages_free(d.table, d.lens, d.ref, none, d.status)
    H.pages_fork(d.pools, d.table, d.lens, d.ref, none, none, 16, d.status)
    H.pages_fork([], d.table, d.lens, d.ref, ints([0]), ints([1]), 16, d.status)          # a fork of nothing: nothing
    H.pages_copy(d.pools, none, none)
    t2, r2 = H.pages_compact([], d.table, d.ref)
    e = torch.empty(0, 2, 8, device="cuda", dtype=torch.float16)
    H.kv_write(e, e, *(torch.zeros(10, 16, 2, 8, device="cuda", dtype=torch.float16) for _ in range(2)), ints([], torch.int64))
    assert all(torch.equal(x, y) for x, y in zip(before, (d.table, d.lens, d.ref))) and int(d.status) == 0
    assert torch.equal(t2, d.table) and torch.equal(r2, d.ref)
    empty = ints([[0] * 4])[:0]
    assert H.pages_extend(empty, none, d.ref, ints([0]), 16, 3, d.status).tolist() == [-1] * 3 and int(d.status) == 0


def test_two_forks_of_one_sequence_and_ends_in_any_order(H):
    """Both forks share the full pages (three references) and own their copies of the last; the pages come free with the last holder."""
    page, pool = 4, torch.randn(12, 4, 5, device="cuda")
    table, lens, ref, status = ints([[-1] * 4] * 4), ints([0] * 4), ints([0] * 12), ints([0])
    H.pages_extend(table, lens, ref, ints([0, 0, 10, 10, 10]), page, 10, status)
    H.pages_fork([pool], table, lens, ref, ints([1, 1]), ints([3, 0]), page, status)
    assert ref.tolist() == [3, 3, 1, 1, 1] + [0] * 7 and lens.tolist() == [10, 10, 0, 10]
    assert table.tolist() == [[0, 1, 4, -1], [0, 1, 2, -1], [-1] * 4, [0, 1, 3, -1]]
    assert torch.equal(pool[3], pool[2]) and torch.equal(pool[4], pool[2])
    H.pages_free(table, lens, ref, ints([1]), status)
    assert ref.tolist() == [2, 2, 0, 1, 1] + [0] * 7
    H.pages_free(table, lens, ref, ints([3, 0]), status)
    assert int(ref.abs().max()) == 0 and int(status) == 0
