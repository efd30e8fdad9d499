"""xdfm_layer_norm_fwd / _bwd at sizes whose passes go past the caches (more than 128 MB), and many rows of a length that
no block's registers hold: out of place against 64 bits, in place with the same bits, gaps between rows left alone."""
import pytest

from tests import test_gpu_layer_norm as base

pytestmark = pytest.mark.gpu

# rows, cols, pad, offset.  16 bits backward: rows of 8 to 32 lanes, in 1, 2, 4 and 8 waves; forward: 8 to 64 lanes, and
# several waves of 16, 24 or 40 elements a lane.
STREAM_16 = [(1700001, 20, 0, 0), (350003, 100, 1, 1), (140001, 250, 0, 0), (70001, 509, 0, 3), (33001, 1000, 0, 0),
             (13100, 2497, 0, 1), (6400, 5113, 3, 0), (3300, 10233, 0, 1), (2100, 16383, 1, 0), (1700, 20477, 0, 0)]
# fp32: rows of 8 to 64 lanes, and in up to 16 waves; 8 waves of many registers backward
STREAM_32 = [(900001, 20, 0, 0), (300001, 61, 1, 1), (140001, 125, 0, 0), (70001, 250, 0, 3), (17001, 1001, 0, 0),
             (7001, 2497, 0, 1), (1400, 12289, 0, 1), (1100, 16381, 1, 0)]


@pytest.mark.parametrize("act", ["identity", "relu", "sigmoid"])
@pytest.mark.parametrize("kind,rows,cols,pad,offset",
                         [(k,) + s for k in ("bf16", "fp16") for s in STREAM_16] + [("fp32",) + s for s in STREAM_32])
def test_passes_past_the_caches(act, kind, rows, cols, pad, offset):
    assert rows * cols * 2 * (4 if kind == "fp32" else 2) > 128e6
    base.test_many_rows_of_a_few_waves_each(act, kind, rows, cols, pad, offset)


@pytest.mark.parametrize("act", ["identity", "relu"])
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,cols,pad,offset", [(533, 20483, 0, 0), (1037, 20489, 3, 1), (4101, 20481, 0, 0)])
def test_many_rows_longer_than_the_registers(act, kind, rows, cols, pad, offset):
    """More rows than the 512 blocks of a launch, and 33, 64 and 256 partial sums of a column."""
    base.test_many_rows_of_a_few_waves_each(act, kind, rows, cols, pad, offset)
