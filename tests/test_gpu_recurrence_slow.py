"""The gated recurrence on the device over gates that remember thousands of steps, so that
every tile of the chained kernels depends on many before it: whole rows against the definition."""

import numpy as np
import pytest

import openpacho as p
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


# Calls whose arrays are more than the last cache holds, and parts of them that are less: accesses past
# the caches and through them have the same bits. Gates of their own, of packed heads and of whole waves.
@pytest.mark.parametrize("sizes,dtype", [((9, 1100, 2048, 2048), np.float32), ((9, 1100, 2048, 256), np.float32), ((9, 1100, 2048, 16), np.float32),
                                         ((900, 20, 1024, 1024), np.float32), ((9, 600, 2048, 2048), np.float64)])  # fmt: skip
def test_gradients_of_more_than_the_last_cache_holds(hip, sizes, dtype):
    print(sizes, dtype, flush=True)
    rows, time, channels, gates = sizes
    rng = p.random.default_rng(1, backend=hip)
    x, d = (rng.normal(0, 1, (rows, time, channels), dtype=dtype) for _ in range(2))
    gate, initial = rng.normal(4, 1, (rows, time, gates), dtype=dtype), rng.normal(0, 1, (rows, channels), dtype=dtype)
    h = p.nn.gated_recurrence(x, gate, initial)
    whole = p.nn.gated_recurrence_grad(d, x, gate, h, initial)
    for part in (slice(0, 2), slice(rows - 2, rows)):
        fewer = p.nn.gated_recurrence_grad(*(a[part] for a in (d, x, gate, h, initial)))
        for one, two in zip(whole, fewer):
            np.testing.assert_array_equal(p.asnumpy(one[part]), p.asnumpy(two))
