"""xdfm_layer_norm_fwd / _bwd on rows that no block's registers hold, up to the longest that are taken.

u = 2^-24, half a step of fp32 relative to the value.
"""
import pytest
import torch

from tests.test_gpu_layer_norm import TYPES, U, bwd, fwd

pytestmark = pytest.mark.gpu


def test_the_weights_gradients_of_more_columns_than_a_launch_has_threads_for():
    """2^27 + 33 columns: 32 threads a column would pass the 2^32 of a launch.  One row, so that dbeta = dy in every bit
    and dgamma = dy (x - mean) rstd after three roundings."""
    cols = (1 << 27) + 33
    dtype, code = TYPES["bf16"]
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((1, cols), generator=gen, device="cuda").to(dtype)
    dy = torch.randn((1, cols), generator=gen, device="cuda").to(dtype)
    one, zero = torch.ones(cols, device="cuda"), torch.zeros(cols, device="cuda")
    stats = torch.tensor([[0.25], [0.75]], device="cuda")
    dx = torch.empty_like(x)
    dg, db = bwd(x, dy, code, one, zero, stats, "identity", dx)
    assert torch.equal(db, dy[0].float())
    exp = dy[0].double() * (x[0].double() - 0.25) * 0.75
    assert ((dg.double() - exp).abs() <= 3 * U * exp.abs() + 2.0 ** -149).all()


@pytest.mark.parametrize("cols", [400001, (1 << 22) + 1, (1 << 27) + 33])
def test_sums_over_equal_terms_do_not_drift(cols):
    """Equal terms round the same way at every addition.  On the way to a row's sum a term passes 3 additions within its
    piece of 4 (those of pieces are 64 bits wide), the rounding to 32 bits, 10 additions over the threads of a block; the
    mean is then divided by the rounded number of columns: 16 u."""
    value = torch.tensor(0.1, device="cuda")
    v, eps = float(value), float(torch.tensor(1e-5))
    one, zero = torch.ones(cols, device="cuda"), torch.zeros(cols, device="cuda")
    x = value.expand(1, cols).contiguous()
    y, stats = torch.empty_like(x), torch.empty((2, 1), device="cuda")
    fwd(x, 0, one, zero, "identity", y, stats, eps=eps)
    assert abs(float(stats[0, 0]) - v) <= 16 * U * v
    # the variance is below 1e-13 of eps; two roundings of the sum with eps and the root, two of the reciprocal
    assert abs(float(stats[1, 0]) * eps ** 0.5 - 1) <= 5 * U
    assert float(y.abs().max()) <= 17 * U * v * float(stats[1, 0])
    # backward: xhat = 1, -1, 1, ... and t = 0.1; mean(t) = 0.1, mean(t xhat) = 0.1 / n
    x[0, 1::2] = -1
    x[0, 0::2] = 1
    stats[0], stats[1] = 0, 1
    dy, dx = value.expand(1, cols).contiguous(), torch.empty_like(x)
    bwd(x, dy, 0, one, zero, stats, "identity", dx)
    exp = -x.double() * (v / cols)
    # 16 u of each of the two means' terms, four roundings of what is added up
    assert float((dx.double() - exp).abs().max()) <= (2 * 16 + 4) * U * v
