"""The attention over the 8-bit cache where its integers, masks and bounds end:
sums of one sign, tokens that a row may not see, rows that see nothing."""
import numpy as np
import pytest

from kv_q8_oracle import PAGE, stored
from test_gpu_kv_q8 import Batch, Cache, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("count", [1, 6, 20])
@pytest.mark.parametrize("pattern", ["flat", "alternating", "random"])
@pytest.mark.parametrize("opposed", [0.0, 0.5, 1.0])
def test_queries_along_and_against_the_keys(gpu, hd, count, pattern, opposed):
    """Every product of a score has the same sign: sums of head_dim * 127 * 128
    and a little less, both ways.  A flat query has the digits -32, -90, 127."""
    rng = np.random.default_rng(hd + count)
    sign = {"flat": np.ones(hd), "alternating": 1.0 - 2.0 * (np.arange(hd) % 2),
            "random": 1.0 - 2.0 * rng.integers(0, 2, hd)}[pattern].astype(np.float32)

    def edit(b):
        b.q[:] = 0.6 * sign
        for x in [b.kp] + b.ks:
            turn = np.where(rng.random((x.shape[0], x.shape[1], 1)) < opposed, -1.0, 1.0)
            x[:] = sign * turn * rng.uniform(0.2, 1.0, (x.shape[0], x.shape[1], 1))
    Batch(gpu, 4, 2, hd, 150, [140], [count], seed=hd, edit=edit).check()
