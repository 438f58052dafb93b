"""Teachers whose logits are large beside their distances, on the device."""

import numpy as np
import pytest

from test_nn_distillation_offsets import OFFSETS, check_offsets

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rest", [True, False])
@pytest.mark.parametrize("vocab", [2, 9, 60, 700, 20000, 70001])
def test_offsets(hip, vocab, rest, dtype):
    for offset, temperature in OFFSETS:
        print(vocab, rest, dtype, offset, temperature, flush=True)
        check_offsets(hip, vocab, dtype, offset, temperature, rest)
