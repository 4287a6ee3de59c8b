"""GPU suite: jb_sample_filtered where its weights and settings are at their limits, against its definition in 64 bits (test_hip_sampler.py)."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_hip_sampler import TYPES, check, definition  # noqa: E402


@pytest.fixture(scope="module")
def H():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from jukebox_amd import _lib, hip_ops
    _lib.lib()          # fail loudly if the extension is missing
    return hip_ops


# Logit x of token 0 (token 1: 0), temperature and u such that u is 1.6e-13 .. 6e-13 of itself beside w / (1 + w), w = exp(x / temp): found by search
# over the floats, among those whose weight lies between two entries of a table of 32 a factor of two.  A weight is a multiple of 2^-44, off by 0.6
# of one: 1.1e-13 of weights from 0.3 on at most.
NEAR = {"f32": ["-0x1.b1ae2cp-5 0x1p+0 0x1.f2735ep-2", "-0x1.b81416p-5 0x1p+0 0x1.f24038p-2", "-0x1.c06ce8p-5 0x1p+0 0x1.f1fd7ep-2",
                "-0x1.32fbe4p-4 0x1p+0 0x1.ecd28ep-2", "-0x1.35563ep-4 0x1p+0 0x1.ecacf6p-2", "-0x1.8f3ed8p-4 0x1p+0 0x1.e71120p-2",
                "-0x1.8f7a1cp-4 0x1p+0 0x1.e70d6ep-2", "-0x1.90c8a8p-4 0x1p+0 0x1.e6f892p-2", "-0x1.4cfed0p-3 0x1p+0 0x1.d67790p-2",
                "-0x1.4d97b2p-3 0x1p+0 0x1.d66494p-2", "-0x1.7945c4p-3 0x1p+0 0x1.d0f94ep-2"],
        "bf16": ["-0x1p+0 0x1.0fa296p+0 0x1.1f232ap-2", "-0x1p+0 0x1.2baacap+0 0x1.31b34ep-2", "-0x1p+0 0x1.bdf1bap+0 0x1.70f274p-2",
                 "-0x1p+0 0x1.d08ff2p+0 0x1.7664ecp-2"],
        "f16": ["-0x1.90c0p-1 0x1.2fe8f6p+0 0x1.5d12b0p-2", "-0x1.90c0p-1 0x1.8910acp+0 0x1.804086p-2", "-0x1.90c0p-1 0x1.891e26p+0 0x1.8044b8p-2",
                "-0x1.90c0p-1 0x1.ae0e9ep+0 0x1.8ad5b4p-2"]}


@pytest.mark.parametrize("dt", sorted(TYPES))
@pytest.mark.parametrize("V", [2, 3000, 20000, 70000])
def test_numbers_next_to_a_border(H, dt, V):
    """The draw, and min-p and top-p at the same weight: on the definition's side of the border, in rows of either size of workgroup."""
    rows = [tuple(float.fromhex(v) for v in r.split()) for t in ("f32", "bf16", "f16") for r in NEAR[t] if t == dt or dt == "f32"]
    x = torch.full((len(rows), V), -math.inf)
    x[:, 0], x[:, 1] = torch.tensor([r[0] for r in rows]), 0.0
    x = x.to(TYPES[dt])
    assert x[:, 0].double().tolist() == [r[0] for r in rows]
    u, temp = (torch.tensor([r[i] for r in rows]) for i in (2, 1))
    for ui, (xi, t, _) in zip(u.tolist(), rows):
        p = 1 / (1 + math.exp(-xi / t))
        assert 1.5e-13 < abs(ui / p - 1) < 1e-12
    check(H, x.cuda(), u, temp)
    # the order is (1, 0): token 0 is kept by top-p if w(1) <= p (w(0) + w(1))
    check(H, x.cuda(), torch.full_like(u, 0.01), temp, p=1 - u)


@pytest.mark.parametrize("V", [40, 30000])
@pytest.mark.parametrize("temp", [1e-45, 1e-38, 1e-30, 3e-20, 1e-10, 1e10, 1e30, 1e37, 3e38, math.inf])
def test_temperatures_of_any_size(H, V, temp):
    """Logits that differ by a few temperatures, however small or large those are: as far as floats go."""
    g = torch.Generator().manual_seed(V)
    t = torch.full((24,), temp)                                        # the float that the row gets
    unit = float(t[0]) if math.isfinite(temp) else 1e38
    x = -torch.rand(24, V, generator=g, dtype=torch.float64) * 40 * unit
    x = torch.clamp(x, -3.4e38, 3.4e38).to(torch.float32)
    x[:, V // 2] = 0.0
    x[::3, 5::7] = -math.inf
    if temp <= 1e-10:                                                  # the largest far from 0 would take the differences' bits
        x[1::3] *= 0.5
        if temp <= 1e-30:                                              # far more temperatures below the largest, all the same near it
            x[2::3, ::2] = (-1e-27 * torch.rand(8, (V + 1) // 2, generator=g, dtype=torch.float64)).to(torch.float32)
            x[2::3, V // 2] = 0.0
    elif temp >= 1e37:                                                 # above and below 0: differences past the largest float
        x[1::3] = ((torch.rand(8, V, generator=g, dtype=torch.float64) - 0.5) * 6.6e38).to(torch.float32)
    u = torch.rand(24, generator=g)
    check(H, x.cuda(), u, t)
    check(H, x.cuda(), u, t, k=7)
    check(H, x.cuda(), u, t, p=0.7)
    for m in (0.05, 0.3, math.exp(-6.3)):
        check(H, x.cuda(), u, t, m=m)
    check(H, x.cuda(), u, t, k=V // 2, p=0.9, m=0.001)


def test_more_rows_than_a_launch_holds(H):
    n = (1 << 24) + 5
    g = torch.Generator("cuda").manual_seed(3)
    x = torch.randn(n, 2, generator=g, device="cuda").half()
    got = H.sample_filtered(x, torch.zeros(n, device="cuda"), 0.0)
    assert torch.equal(got, (x[:, 1] > x[:, 0]).long())


@pytest.mark.parametrize("dt,V,n", [("f32", 300, 5000), ("bf16", 17000, (1 << 22) + 3), ("f16", 2048, 1)])
def test_one_row_drawn_from_many_times(H, dt, V, n):
    """A row expanded to n of them (a pitch of 0), each with a number and a temperature of its own."""
    g = torch.Generator("cuda").manual_seed(V)
    # two temperatures: at 0.5 the weights of these logits are squares of those at 1
    row = torch.randint(0, 12, (1, V), generator=g, device="cuda").double()
    x = (row * math.log(2.0)).to(TYPES[dt])
    u = torch.rand(n, generator=g, device="cuda")
    temp = torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, 0.5, 1.0)
    got = H.sample_filtered(x.expand(n, V), u, temp)
    for t in (0.5, 1.0):
        rows = temp == t
        if not bool(rows.any()):
            continue
        w = torch.exp((x[0].double() - x.double().max()) / t)
        cum = torch.cumsum(w, 0)
        goal = u[rows].double() * cum[-1]
        # (rows whose number falls onto a border, to the two sums' own rounding, are left out)
        i = torch.searchsorted(cum, goal, right=True)
        near = torch.minimum((cum[i] - goal).abs(), (goal - torch.where(i > 0, cum[(i - 1).clamp(min=0)], goal - 1)).abs()) < 1e-9 * cum[-1]
        assert bool(((got[rows] == i) | near).all()) and float(near.double().mean()) < 1e-3
    if n > 1000:
        full = x.expand(1000, V).contiguous()
        assert torch.equal(got[:1000], H.sample_filtered(full, u[:1000].contiguous(), temp[:1000].contiguous()))
        assert torch.equal(got[-1000:], H.sample_filtered(full, u[-1000:].contiguous(), temp[-1000:].contiguous()))


def test_equal_logits_at_the_border_of_two_samplers(H):
    """Four equal logits and top-k 2: jb_sample_logits draws from all four, as a threshold keeps them; this from the two lowest indices."""
    n = 256
    x = torch.full((n, 64), -3.0, device="cuda")
    x[:, [7, 20, 33, 50]] = 1.0
    tokens, t_dev = torch.zeros(n, 1, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    H.sample_logits(x, H.make_sample_params(top_k=2, seed=5), tokens, t_dev)
    assert set(tokens[:, 0].tolist()) == {7, 20, 33, 50}
    assert set(H.sample_filtered(x, torch.rand(n, device="cuda"), top_k=2).tolist()) == {7, 20}
