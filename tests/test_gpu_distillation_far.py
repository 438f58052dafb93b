"""A rest far below the listed logits, on the device: in rows of every team and of several pieces."""

import numpy as np
import pytest

from test_nn_distillation_far import GAPS, VOCABULARIES, check_far_rest, check_far_rest_by_hand, check_nothing_left

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("vocab", VOCABULARIES + [1000, 3000, 8193, 20000, 40003, 90001])
def test_far_rest(hip, vocab, dtype):
    for gap in GAPS if vocab < 3000 else (80, 100, 1000):
        print(vocab, gap, dtype, flush=True)
        check_far_rest(hip, vocab, dtype, gap)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_far_rest_by_hand(hip, dtype):
    check_far_rest_by_hand(hip, dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("vocab", [5, 70, 700, 9000, 70001])
def test_nothing_left(hip, vocab, dtype):
    check_nothing_left(hip, dtype, vocab)
