"""xdfm_layer_norm_fwd / _bwd at values where their arithmetic can go wrong: rows that are not finite, sums whose order
shows, activations far out.

u = 2^-24, half a step of fp32 relative to the value.
"""
import pytest
import torch

from tests.test_gpu_layer_norm import ACT, TYPES, U, bwd, fwd, half_step, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_row_that_is_not_finite_reads_as_nan_under_every_activation(act, kind, bad):
    """One NaN or infinity leaves a row without a mean: it has no values, and zeros would hide that."""
    dtype, code = TYPES[kind]
    for rows, cols in ((40, 5), (40, 20), (40, 1024), (33, 2496), (20, 9000), (3, 30001)):
        x, _, gamma, beta, _ = make(rows, cols, dtype, seed=cols)
        y, y2 = torch.empty_like(x), torch.empty_like(x)
        stats = torch.empty((2, rows), device="cuda")
        fwd(x, code, gamma, beta, act, y, stats)
        assert torch.isfinite(y).all()
        x[1, cols // 2] = bad
        fwd(x, code, gamma, beta, act, y2, stats)
        assert torch.isnan(y2[1]).all()
        keep = [r for r in range(rows) if r != 1]
        assert torch.equal(y2[keep], y[keep])


def test_the_join_of_partial_sums_does_not_lose_small_ones():
    """8192 x 20: a row's dy of 1 and 31 of 2^-24 in rows 64, 128, ..., which lie in partial sums of their own.  Half a
    step under 1 each, they are lost where all 32 are added to the 1 one after the other: 31 u.  In a tree the 1 passes 5
    additions of the join, and before it 7 within a block (8 groups of a wave, 8 waves and its own row) and 3 of the 4
    parts of a slice: 15 u of 1 at most, and the small ones' own additions are exact."""
    rows, cols = 8192, 20
    x = torch.zeros((rows, cols), device="cuda")
    dy = torch.zeros((rows, cols), device="cuda")
    dy[0] = 1
    dy[64:2048:64] = 2.0 ** -24
    one, zero = torch.ones(cols, device="cuda"), torch.zeros(cols, device="cuda")
    stats = torch.zeros((2, rows), device="cuda")
    stats[0], stats[1] = -1, 1  # xhat = 1: dgamma is the same sum
    dg, db = bwd(x, dy, 0, one, zero, stats, "identity", torch.empty_like(x))
    exp = 1 + 31 * 2.0 ** -24
    for got in (dg, db):
        assert ((got.double() - exp).abs() <= 15 * U).all(), float((got.double() - exp).abs().max()) / U


def far_out(cols):
    """u of a row: over +-120, near 0, and next to where the forms change or exponentials leave their range."""
    gen = torch.Generator(device="cuda").manual_seed(cols)
    u = torch.empty(cols, device="cuda").uniform_(-120, 120, generator=gen)
    small = torch.empty(cols, device="cuda").uniform_(-20, 1.5, generator=gen).exp()
    u[1::3] = (small * torch.sign(u))[1::3]
    edge = torch.tensor([0.0, 0.1, 0.5, 0.6, 87.3, 87.4, 88.0, 88.7, 88.8, 103.0, 104.0, 119.0], device="cuda")
    edge = torch.cat([edge, edge * (1 + 2.0 ** -22), edge * (1 - 2.0 ** -22)])
    edge = torch.cat([edge, -edge])
    u[:edge.numel()] = edge
    return u


def activation(act, u):
    """Value and slope in 64 bits."""
    if act == "sigmoid":
        return torch.sigmoid(u), 0.25 / torch.cosh(u / 2) ** 2
    if act == "tanh":
        return torch.tanh(u), 1 / torch.cosh(u) ** 2
    return torch.where(u > 0, u, torch.expm1(u)), torch.where(u > 0, torch.ones_like(u), torch.exp(u))


# The hardware's 2^x and reciprocal are good to one unit of the last place, 2 u.
#
# fp32 results.  sigmoid = 1 / (1 + e): e to 3.1 u (2^x, and the rounding that puts back what the product cut off), the
# addition and the reciprocal 3 u: 6.1.  tanh from 0.6 on = 1 - 2 / (e + 1), e to (2 + 2.45 |u|) u (2^x of a rounded
# product with a rounded constant): (1 - t)(5 + 2.45 |u|) + t units, 6.6 t at 0.6 and less beyond; below 0.6 the series
# is good to 2 u.  elu from -0.5 down = e - 1, e to (2 + 1.23 |u|) u: 2 units at -0.5, 5.1 of the value, and less beyond.
# Results of 16 bits, before they are stored.  sigmoid: e to (2 + 1.23 |u|) u, 3 u more.  tanh from 0.1 on as above: 4.9
# units of 0.0997, 49 of the value; elu from -0.1 down 2.1 units of 0.095, 22; their series below that: 4 and 16.
VALUE = {("sigmoid", 4): lambda u: 6.2, ("tanh", 4): lambda u: 7.0, ("elu", 4): lambda u: 6.0,
         ("sigmoid", 2): lambda u: 5 + 1.3 * u.abs(), ("tanh", 2): lambda u: 50.0, ("elu", 2): lambda u: 24.0}
# Slopes, in units of 1, the same for every type.  s (1 - s): s |1 - 2 s| times what s is off by, two roundings: 6.6 at
# most.  1 - t t: 2 t times what t is off by, two roundings: 3.9 + 1.6 near u = 1, less elsewhere.  e^u: 3.1.
SLOPE = {"sigmoid": 6.6, "tanh": 6.0, "elu": 3.2}


@pytest.mark.parametrize("rows,cols", [(1, 1000), (1030, 1000), (300, 9000), (2, 40001)])
@pytest.mark.parametrize("act", list(SLOPE))
@pytest.mark.parametrize("kind", list(TYPES))
def test_activations_far_out(kind, act, rows, cols):
    """Rows of zeros have xhat = 0, so u = beta in every bit: results, and slopes as the dbeta of one row of ones."""
    dtype, code = TYPES[kind]
    u = far_out(cols)
    x, one = torch.zeros((rows, cols), dtype=dtype, device="cuda"), torch.ones(cols, device="cuda")
    y, stats = torch.empty_like(x), torch.empty((2, rows), device="cuda")
    fwd(x, code, one, u, act, y, stats)
    value, slope = activation(act, u.double())
    size = x.element_size()
    off = VALUE[act, size](u.double()) * U * value.abs() + 2.0 ** -125  # (the reciprocal has no denormal results)
    if size == 2:  # stored: half a step of the type (u itself was counted above for fp32)
        off = off + half_step(dtype, value.abs() + off)
    err = (y.double() - value).abs()
    assert (err <= off).all(), float((err / off).max())
    dy = torch.zeros_like(x)
    dy[rows - 1] = 1
    dg, db = bwd(x, dy, code, one, u, stats, act, torch.empty_like(x))
    err = (db.double() - slope).abs()
    assert (err <= SLOPE[act] * U + 2.0 ** -125).all(), float(err.max() / U)
    assert (dg == 0).all()
