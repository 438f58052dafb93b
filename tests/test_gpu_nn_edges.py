"""Operators of ``nn`` on the device at the ends of what they take."""

import numpy as np
import pytest

from test_nn_adamw import check_mixed_lists
from test_nn_losses import check_impossible_responses, check_impossible_tokens, check_near_policies

pytestmark = pytest.mark.gpu


def test_mixed_lists(hip):
    check_mixed_lists(hip)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_impossible_responses(hip, dtype):
    check_impossible_responses(hip, dtype)


# Short rows, rows of one workgroup, rows in pieces.
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("vocab", [2, 40, 3000, 70001])
def test_impossible_tokens(hip, vocab, dtype):
    check_impossible_tokens(hip, dtype, vocab)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_near_policies(hip, dtype):
    check_near_policies(hip, dtype)
