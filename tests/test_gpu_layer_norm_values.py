"""xdfm_layer_norm_fwd / _bwd at values where their arithmetic can go wrong: rows that are not finite, sums whose order
shows, activations far out.

u = 2^-24, half a step of fp32 relative to the value.
"""
import pytest
import torch

from tests.test_gpu_layer_norm import ACT, TYPES, U, bwd, fwd, make

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
