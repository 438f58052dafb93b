"""``nn.distillation_loss`` of lists that name an index again and go on with others, on the NumPy backend."""

import numpy as np
import pytest

import openpacho as p
from oracle import blocks
from test_nn_losses import put, within

FLOATS = [np.float32, np.float64]
# (vocabulary, entries, distinct names): more entries than the lanes of any team that works on a list, 4 to 64.
LISTS = [(10, 12, 6), (20, 40, 11), (40, 60, 25), (100, 90, 50), (250, 140, 90), (3000, 200, 120), (20000, 150, 100), (90001, 1024, 700)]


def check_repeats_in_long_lists(backend, vocab, entries, names, dtype, rows=5):
    """Every name comes once among the first entries or after a repeat; half of the rest of the list are repeats."""
    rng = np.random.default_rng(vocab)
    z = rng.standard_normal((rows, vocab)).astype(dtype)
    order = np.empty((rows, entries), np.int64)
    for row in range(rows):
        distinct = rng.permutation(vocab)[:names]
        again = np.zeros(entries, bool)
        again[1 + rng.permutation(entries - 1)[: entries - names]] = True
        order[row, ~again] = distinct
        for entry in np.flatnonzero(again):
            order[row, entry] = order[row, rng.integers(0, entry)]
    listed, rest = rng.standard_normal((rows, entries)).astype(dtype), rng.standard_normal(rows).astype(dtype)
    for others in (rest, None):
        values, units = blocks.distillation_loss(z, order, listed, others, temperature=1.25)
        given = put(backend, z, order, listed, others)
        found = p.nn.distillation_loss_grad(*given, temperature=1.25)
        for got, want, unit in zip(found, values, units):
            within(got, want, unit, dtype)
        for got, same in zip(p.nn.distillation_loss(*given, temperature=1.25), found):
            np.testing.assert_array_equal(p.asnumpy(got), p.asnumpy(same))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("vocab,entries,names", LISTS[:-1])
def test_repeats_in_long_lists(numpy_backend, vocab, entries, names, dtype):
    check_repeats_in_long_lists(numpy_backend, vocab, entries, names, dtype)
