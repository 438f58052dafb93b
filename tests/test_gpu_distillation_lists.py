"""Lists that name an index again, on the device: by teams of every size and by pieces of rows."""

import numpy as np
import pytest

from test_nn_distillation_lists import LISTS, check_repeats_in_long_lists

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("vocab,entries,names", LISTS)
def test_repeats_in_long_lists(hip, vocab, entries, names, dtype):
    print(vocab, entries, names, dtype, flush=True)
    check_repeats_in_long_lists(hip, vocab, entries, names, dtype)
