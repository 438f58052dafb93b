"""The gated recurrence on the device over gates that remember thousands of steps, so that
every tile of the chained kernels depends on many before it: whole rows against the definition."""

import numpy as np
import pytest

from test_nn_recurrence import check_slow

pytestmark = pytest.mark.gpu

# Tiles have 128 steps forward and 64 backward (64 and 32 of float64). Blocks of 64 tiles below 32 groups
# of channels and of 16 from there on, several of each: gates of their own, heads that share a wave, heads of
# whole waves, heads in pieces of waves.
SIZES = [(1, 17000, 70, 70), (1, 17000, 60, 12), (1, 17000, 128, 2), (1, 17000, 100, 1), (2, 2200, 1030, 1030), (1, 2200, 2048, 16),
         (1, 2200, 2048, 256), (2, 2200, 990, 30)]  # fmt: skip


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("resets", [False, True])
@pytest.mark.parametrize("sizes", SIZES)
def test_slow_gates(hip, sizes, resets, dtype):
    print(sizes, resets, dtype, flush=True)
    check_slow(hip, sizes, dtype, resets)


# The kernels of rows that are no tiles: one wave, four, eight and two runs of these.
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("time", [1, 3, 16, 60, 128, 250])
def test_slow_gates_of_shorter_rows(hip, time, dtype):
    check_slow(hip, (3, time, 66, 6), dtype, False)
    check_slow(hip, (2, time, 70, 70), dtype, True)
