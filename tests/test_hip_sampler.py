"""GPU suite: jb_sample_filtered against its definition in 64 bits (numpy).  The answers are whole numbers and have to be equal:
the definition's own border cases (u times the total against a partial sum, a weight sum against top-p) are met only by chance of
some 10^-11 a row with these inputs, apart from those made to fall exactly on one."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def H():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from jukebox_amd import _lib, hip_ops
    _lib.lib()          # fail loudly if the extension is missing
    return hip_ops


def definition(x, u, temp, k, p, m):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return -1
    if not temp > 0:
        return int(np.argmax(x))
    order = np.argsort(-x, kind="stable")
    if k > 0:
        order = order[:k]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / np.float64(temp)))
    w[x[order] == -np.inf] = 0.0                       # forbidden whatever the temperature (-inf / inf is no number)
    if 0 < p < 1:
        keep = np.concatenate([[0.0], np.cumsum(w)[:-1]]) <= np.float64(p) * w.sum()
        order, w = order[keep], w[keep]
    if m > 0:
        keep = w >= min(np.float64(m), 1.0)
        order, w = order[keep], w[keep]
    by = np.argsort(order)
    order, cum = order[by], np.cumsum(w[by])
    live = np.flatnonzero(w[by])
    return int(order[min(np.searchsorted(cum, np.float64(max(u, 0.0)) * cum[-1], side="right"), live[-1])])


def check(H, x, u, temp=1.0, k=0, p=0.0, m=0.0):
    R = x.shape[0]
    full = lambda v, t: torch.full((R,), v, dtype=t) if not torch.is_tensor(v) else v.to(t)  # noqa: E731
    temp, k, p, m = full(temp, torch.float32), full(k, torch.int32), full(p, torch.float32), full(m, torch.float32)
    got = H.sample_filtered(x, u.cuda(), temp.cuda(), k.cuda(), p.cuda(), m.cuda()).tolist()
    rows = x.float().cpu().numpy()
    want = [definition(rows[i], *(float(v[i]) for v in (u, temp)), int(k[i]), float(p[i]), float(m[i])) for i in range(R)]
    bad = [(i, g, w) for i, (g, w) in enumerate(zip(got, want)) if g != w]
    assert not bad, f"(row, got, want): {bad[:5]}, {len(bad)} of {R}; settings of the first: {[float(v[bad[0][0]]) for v in (u, temp, k, p, m)]}"


def logits(R, V, dt, seed, spread=2.5):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(R, V, generator=g, device="cuda") * spread
    x[torch.rand(R, V, generator=g, device="cuda") < 0.05] = -math.inf
    return x.to(TYPES[dt]), torch.rand(R, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dt", sorted(TYPES))
@pytest.mark.parametrize("V", [1, 2, 7, 64, 80, 1000, 2048, 4111, 50001, 128000, 262144])
@pytest.mark.parametrize("what", ["none", "k", "p", "m", "kp", "all"])
def test_filters(H, dt, V, what):
    R = 24 if V < 50000 else 8
    x, u = logits(R, V, dt, V)
    rng = np.random.default_rng(V)
    pick = lambda *v: torch.tensor([v[rng.integers(len(v))] for _ in range(R)])  # noqa: E731
    kw = {"temp": pick(0.3, 0.7, 1.0, 1.5)}
    if what in ("k", "kp", "all"):
        kw["k"] = pick(1, 2, 40, 500, 1500, V, V + 3)
    if what in ("p", "kp", "all"):
        kw["p"] = pick(0.01, 0.5, 0.9, 0.99, 0.9999)
    if what in ("m", "all"):
        kw["m"] = pick(0.001, 0.05, 0.5, 1.0, 2.0)
    check(H, x, u, **kw)


def test_one_number_for_all_rows_and_defaults(H):
    x, u = logits(16, 3000, "f32", 1)
    n = lambda v, t=torch.float32: torch.full((16,), v, dtype=t, device="cuda")  # noqa: E731
    assert torch.equal(H.sample_filtered(x, u.cuda(), 0.8, 50, 0.9, 0.01), H.sample_filtered(x, u.cuda(), n(0.8), n(50, torch.int32), n(0.9), n(0.01)))
    assert torch.equal(H.sample_filtered(x, u.cuda()), H.sample_filtered(x, u.cuda(), n(1.0), n(0, torch.int32), n(0.0), n(0.0)))
    out = torch.zeros(16, dtype=torch.int64, device="cuda")
    assert H.sample_filtered(x, u.cuda(), out=out) is out and torch.equal(out, H.sample_filtered(x, u.cuda()))


@pytest.mark.parametrize("dt", sorted(TYPES))
def test_equal_logits(H, dt):
    """Rows of few distinct values: ties go to the lowest index, in the order and so in the filters."""
    for V in (5, 1024, 1025, 5000, 70000):
        g = torch.Generator("cuda").manual_seed(V)
        x = torch.randint(0, 3, (12, V), generator=g, device="cuda").to(TYPES[dt])
        x[0] = 1.0
        x[1] = 0.0
        x[1, ::2] = -0.0
        u = torch.rand(12, generator=torch.Generator().manual_seed(V))
        check(H, x, u)
        check(H, x, u, k=torch.tensor([1, 2, 3, 4, V // 2, V // 2, V - 1, V, 1, 2, 3, V // 3]))
        check(H, x, u, p=torch.linspace(0.05, 0.97, 12))
        check(H, x, u, k=max(1, V // 3), p=torch.linspace(0.05, 0.97, 12), m=0.2)


def test_borders_met_exactly(H):
    """Four equal logits: every sum is a whole number of quarters, and u, p fall on them."""
    x = torch.zeros(9, 4, device="cuda")
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.249999, 0.999999, 0.5, 0.0, 0.75])
    check(H, x, u)
    check(H, x, u, p=0.5)
    check(H, x, u, p=0.25)
    check(H, x, u, p=0.75, k=3)
    check(H, x, u, m=1.0)
    got = H.sample_filtered(x, torch.tensor([1.0, 2.0, math.inf, -1.0, math.nan, 0.5, 0.0, 0.0, 0.0], device="cuda"))
    assert got.tolist() == [3, 3, 3, 0, 0, 2, 0, 0, 0]


@pytest.mark.parametrize("dt", sorted(TYPES))
def test_forbidden_tokens(H, dt):
    low = torch.finfo(TYPES[dt]).min
    x = torch.zeros(8, 600, device="cuda")
    x[0] = -math.inf                                   # nothing allowed
    x[1] = math.nan
    x[2] = -math.inf
    x[2, 577] = -3.0                                   # one allowed
    x[3] = low                                         # a mask of the type's lowest value everywhere: all are equal
    x[4] = low
    x[4, 5], x[4, 590] = 1.0, 1.5
    x[5, ::2] = math.nan
    x[6] = -math.inf
    x[6, 17], x[6, 400] = math.inf, math.inf           # infinitely likely: only they
    x[7, 3] = math.inf
    x = x.to(TYPES[dt])
    for u in (0.0, 0.3, 0.9):
        for kw in ({}, {"k": 2}, {"p": 0.6}, {"m": 0.5}, {"temp": 0.0}, {"temp": 1e-30}, {"k": 100, "p": 0.9, "m": 0.01}):
            check(H, x, torch.full((8,), u), **kw)
    assert H.sample_filtered(x, torch.zeros(8, device="cuda")).tolist()[:2] == [-1, -1]


def test_temperatures(H):
    x, u = logits(14, 5000, "f32", 7)
    check(H, x, u, temp=torch.tensor([0.0, -1.0, 1e-6, 1e-3, 0.05, 0.1, 0.99, 1.0, 5.0, 50.0, 1e4, 1e20, math.inf, math.nan]))
    check(H, x, u, temp=torch.tensor([0.0, -1.0, 1e-6, 1e-3, 0.05, 0.1, 0.99, 1.0, 5.0, 50.0, 1e4, 1e20, math.inf, math.nan]), k=60, p=0.95)


def test_logits_far_apart(H):
    """Values over the whole range of the type, so that nearly all weights vanish."""
    for dt, hi in (("f32", 1e30), ("f16", 6e4), ("bf16", 1e30)):
        x, u = logits(8, 4000, dt, 9)
        x = (x.float() * (hi / 20)).to(TYPES[dt])
        check(H, x, u, k=30)
        check(H, x, u, p=0.9)
        check(H, x, u)


def test_pitch_and_untouched_neighbours(H):
    wide = torch.randn(6, 3, 1001, device="cuda").half()
    x = wide[:, 1, 3:1000]
    u = torch.rand(6)
    want = H.sample_filtered(x.contiguous(), u.cuda(), top_p=0.9)
    assert torch.equal(H.sample_filtered(x, u.cuda(), top_p=0.9), want)
    assert H.sample_filtered(x[:0], u.cuda()[:0]).shape == (0,)


def test_many_rows_and_frequencies(H):
    """One row drawn from often: the frequencies are the probabilities' (five standard deviations)."""
    N, V = 20000, 12
    x = torch.randn(1, V, generator=torch.Generator().manual_seed(5)).cuda()
    u = torch.rand(N, generator=torch.Generator().manual_seed(6)).cuda()
    got = H.sample_filtered(x.expand(N, V).contiguous(), u, temp=0.9)
    p = torch.softmax(x[0].double() / 0.9, 0).cpu().numpy()
    f = np.bincount(got.cpu().numpy(), minlength=V) / N
    assert np.all(np.abs(f - p) < 5 * np.sqrt(p * (1 - p) / N))


def test_agrees_with_the_step_sampler(H):
    """jb_sample_logits with its own generator: greedy and top_k = 1 pick the same tokens."""
    x, u = logits(16, 2048, "f32", 11)
    x = torch.where(x == -math.inf, -100.0, x)
    params = H.make_sample_params(temp=0.99, top_k=1)
    tokens, t_dev = torch.zeros(16, 4, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    H.sample_logits(x, params, tokens, t_dev)
    assert torch.equal(tokens[:, 0], H.sample_filtered(x, u.cuda(), temp=0.99, top_k=1))
    assert torch.equal(tokens[:, 0], H.sample_filtered(x, u.cuda(), temp=0.0))


def test_in_a_graph(H):
    x, u = logits(32, 9000, "bf16", 13)
    u = u.cuda()
    p = torch.full((32,), 0.9, device="cuda")
    out = torch.zeros(32, dtype=torch.int64, device="cuda")
    H.sample_filtered(x, u, 0.8, 0, p, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        H.sample_filtered(x, u, 0.8, 0, p, out=out)
    for step in range(3):
        u.copy_(torch.rand(32, generator=torch.Generator().manual_seed(step)))
        p.fill_(0.5 + 0.1 * step)
        want = H.sample_filtered(x, u, 0.8, 0, p)
        torch.cuda.synchronize()
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_settings_as_large_as_they_may_be(H):
    x, u = logits(4, 500, "f32", 31)
    u = u.cuda()
    want = H.sample_filtered(x, u)
    for k in (500, 2 ** 31 - 1, 2 ** 40, -1, -2 ** 40):          # all of them, or off
        assert torch.equal(H.sample_filtered(x, u, top_k=k), want)
    assert torch.equal(H.sample_filtered(x, u, top_p=7.0), want) and torch.equal(H.sample_filtered(x, u, min_p=-3.0), want)
    assert torch.equal(H.sample_filtered(x, u, min_p=9.0), x.argmax(1)) and torch.equal(H.sample_filtered(x, u, top_k=1), x.argmax(1))
    assert H.sample_filtered(x[:0], u[:0]).numel() == 0
    assert H.sample_filtered(x, u, temp=math.inf).min() >= 0


def test_two_streams_at_once(H):
    (x, u), (y, v) = logits(64, 128000, "bf16", 32), logits(300, 2048, "f32", 33)
    u, v = u.cuda(), v.cuda()
    want = [H.sample_filtered(x, u, 0.9, 50, 0.9), H.sample_filtered(y, v, 1.0, 0, 0.9)]
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        with torch.cuda.stream(s):
            outs[0].append(H.sample_filtered(x, u, 0.9, 50, 0.9))
        with torch.cuda.stream(t):
            outs[1].append(H.sample_filtered(y, v, 1.0, 0, 0.9))
    torch.cuda.synchronize()
    assert all(torch.equal(w, o) for w, os in zip(want, outs) for o in os)
