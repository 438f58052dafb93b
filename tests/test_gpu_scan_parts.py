"""The selective scan on the device where a row's parts meet more states than a launch takes, and of calls on both sides of
the number of workgroups from which rows stay whole."""

import numpy as np
import pytest

from test_nn_blocks import check_scan

pytestmark = pytest.mark.gpu


# Sixteen waves forward, and two or more launches over the states that use a row's parts again.
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("full,resets,lengths", [(True, True, True), (True, False, False), (False, False, True)])
@pytest.mark.parametrize("sizes", [(1, 700, 20, 1, 64), (1, 300, 5, 1, 40), (1, 300, 5, 1, 130)])
def test_many_states_in_parts(hip, sizes, full, resets, lengths, dtype):
    print(sizes, full, resets, lengths, dtype, flush=True)
    check_scan(hip, sizes, dtype, full, resets, lengths, seed=3)


# 128 workgroups in parts; 129, 150 and 255 whole.
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("sizes", [(128, 70, 3, 1, 4), (129, 70, 3, 1, 4), (75, 70, 70, 1, 3), (85, 65, 3, 3, 16)])
def test_workgroups(hip, sizes, dtype):
    print(sizes, dtype, flush=True)
    check_scan(hip, sizes, dtype, True, True, True, seed=4)
