"""What joins gate and up behind products in 8-bit integers, by itself: sums and scales are chosen so that both floats are exact (whole numbers
of at most 2 * 127 * 127 times powers of two), and the gate's own error is what is left.

In float32, unit 2^-24 of the result: an exponential of two units in the last place (4), a sum, a quotient and the product with up (1 each) make 7,
and one is left for what is smaller; behind alpha, or the polynomial of the tanh gelu (7 roundings), the exponent is off by one rounding of itself, or
by 7, and the gate with it, by as much as its exponential counts.  Below an exponent of -87 the exponential leaves the floats and the result
is 0 (by itself it would be below 2e-36 times up).
"""
import pytest
import torch

import test_int8_gpu as T

pytestmark = pytest.mark.gpu
GATES = [("silu", 0.0, 1.0), ("gelu_tanh", 0.0, 1.0), ("clamped_swish", 7.0, 2.0), ("clamped_swish", 3.0, 1.702)]
# one to 16 tokens; single tiles; clusters of two and of four that share k; pairs
SIZES = [(1, 700, 600), (5, 300, 512), (16, 129, 400), (20, 640, 512), (130, 1024, 304), (30, 96, 2048), (64, 520, 2048), (128, 1024, 8192), (2100, 4096, 512)]


def parts(tokens, n, k):
    """(rows, weight, gate, up): the last two in 64 bits, exact in float."""
    m = T.int8()
    g = torch.Generator().manual_seed(tokens + n)
    rows = torch.zeros(tokens, m.row_pitch(k), dtype=torch.int8)
    w = torch.zeros(2 * n, m.row_pitch(k), dtype=torch.int8)
    for at in (0, k // 2 + 3):
        rows[:, at] = torch.randint(-127, 128, (tokens,), generator=g, dtype=torch.int8)
        w[:, at] = torch.randint(-127, 128, (2 * n,), generator=g, dtype=torch.int8)
    s = 2.0 ** -torch.randint(4, 8, (tokens,), generator=g).float()
    c = 2.0 ** -torch.randint(4, 9, (2 * n,), generator=g).float()
    y = (rows.double() @ w.double().t()) * s.double()[:, None] * c.double()
    y = y.to(T.DEV)
    return m.Int8Rows(rows.to(T.DEV)[:, :k], s.to(T.DEV)), m.Int8Weight(w.to(T.DEV)[:, :k], c.to(T.DEV)), y[:, :n], y[:, n:]


def definition(gate, up, glu, limit, alpha):
    """(the result, the gate's exponent, how far its roundings move it, in units) in 64 bits."""
    if glu == "silu":
        x, off = gate, 0.0
    elif glu == "gelu_tanh":
        x, off = 1.5957691216057307 * (gate + 0.044715 * gate ** 3), 7.0          # (tanh(z) = 2 sigmoid(2 z) - 1)
    else:
        alpha = float(torch.tensor(alpha, dtype=torch.float32))
        gate, up = gate.clamp_max(limit), up.clamp(-limit, limit) + 1.0
        x, off = alpha * gate, 1.0
    return gate * torch.sigmoid(x) * up, x, off * x.abs() * torch.sigmoid(-x)


@pytest.mark.parametrize("glu,limit,alpha", GATES)
@pytest.mark.parametrize("tokens,n,k", SIZES)
def test_a_gate_in_float32(tokens, n, k, glu, limit, alpha):
    rows, w, gate, up = parts(tokens, n, k)
    got = T.int8().int8_glu(rows, w, glu=glu, limit=limit, alpha=alpha, out_dtype=T.F32).double()
    want, x, off = definition(gate, up, glu, limit, alpha)
    near = x >= -87.0
    assert tokens == 1 or near.float().mean() > 0.6 and (near & (x < -12.0)).any()       # (one token's gates are as large as it drew them)
    tol = (8.0 + off) * 2.0 ** -24 * want.abs() + 1e-44
    bad = near & ~((got - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / tol)[near].max()))
    assert (got - want).abs()[~near].le((2e-36 * (up.abs() + 1.0))[~near]).all()


@pytest.mark.parametrize("glu,limit,alpha", GATES)
@pytest.mark.parametrize("tokens", [1, 12, 40, 300])
@pytest.mark.parametrize("out_dtype", [T.BF16, T.F32])
def test_a_gate_of_what_is_no_number(tokens, glu, limit, alpha, out_dtype):
    """Infinite and missing sums (a scale that is infinite or NaN), and sums of zero: what the formula gives of them in floats."""
    m = T.int8()
    inf, nan = float("inf"), float("nan")
    gates, ups = torch.tensor([inf, -inf, nan, 0.0, 1.0, 1.0, 1.0, 1e30, -1e30]), torch.tensor([2.0, 2.0, 2.0, 3.0, inf, nan, 0.0, 2.0, 2.0])
    rows = m.Int8Rows(torch.ones(tokens, 16, dtype=torch.int8, device=T.DEV)[:, :1], torch.ones(tokens, device=T.DEV))
    values = torch.ones(18, 16, dtype=torch.int8, device=T.DEV)[:, :1]
    got = m.int8_glu(rows, m.Int8Weight(values, torch.cat([gates, ups]).to(T.DEV)), glu=glu, limit=limit, alpha=alpha, out_dtype=out_dtype)
    g, u = gates.double(), ups.double()
    want = T.gated(torch.stack([g, u]).reshape(1, -1), glu, limit, alpha)[0]
    clamped = glu == "clamped_swish"
    # (an infinity times a factor of zero has no value; behind a limit plus infinity is the limit)
    lost = torch.tensor([False, True, True, False, False, True, False, False, False])
    got = got.double().cpu()
    assert torch.equal(got.isnan(), lost.expand(tokens, -1)), got[0]
    for at in range(9):
        if lost[at]:
            continue
        if want[at].isinf():
            assert (got[:, at] == want[at]).all(), (at, got[0, at], want[at])
        else:
            assert ((got[:, at] - want[at]).abs() <= 2.0 ** -8 * want[at].abs() + 1e-30).all(), (at, got[0, at], want[at], clamped)
