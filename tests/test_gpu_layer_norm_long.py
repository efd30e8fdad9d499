"""xdfm_layer_norm_fwd / _bwd on rows that no block's registers hold, up to the longest that are taken.

u = 2^-24, half a step of fp32 relative to the value.
"""
import pytest
import torch

from tests.test_gpu_layer_norm import TYPES, U, bwd

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
