"""States that forget at once, on the device: behind rows' ends and in the steps that fill a tile, in groups that leave
lanes without a channel, and in parts of rows."""

import pytest

from test_nn_scan_rates import FLOATS, RATES, SIZES, check_no_rate, check_rates, check_rates_of_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("sizes", SIZES + [(1, 40, 70, 1, 33), (1, 150, 5, 1, 4), (2, 300, 66, 2, 16), (1, 200, 3, 1, 70)])
def test_rates(hip, sizes, dtype):
    for a_log in RATES[dtype]:
        print(sizes, a_log, dtype, flush=True)
        check_rates(hip, sizes, dtype, a_log)


@pytest.mark.parametrize("dtype", FLOATS)
def test_rates_of_tokens(hip, dtype):
    check_rates_of_tokens(hip, dtype)
    check_rates_of_tokens(hip, dtype, (2, 1, 130, 1, 40))


@pytest.mark.parametrize("dtype", FLOATS)
def test_no_rate(hip, dtype):
    check_no_rate(hip, dtype)
