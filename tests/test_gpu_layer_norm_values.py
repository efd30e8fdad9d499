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
