"""Carried states and gradients near the type's ends, in parts of rows on the device."""

import pytest

from test_nn_scan_large_states import FLOATS, check_infinite_states, check_large_states

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("sizes", [(1, 400, 3, 1, 3), (2, 700, 20, 2, 16), (1, 300, 70, 1, 20), (1, 300, 5, 1, 40)])
def test_large_states(hip, sizes, dtype):
    print(sizes, dtype, flush=True)
    check_large_states(hip, sizes, dtype)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("sizes", [(1, 400, 3, 1, 3), (2, 700, 20, 2, 16), (1, 300, 5, 1, 40)])
def test_infinite_states(hip, sizes, dtype):
    print(sizes, dtype, flush=True)
    check_infinite_states(hip, sizes, dtype)
