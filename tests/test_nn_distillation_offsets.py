"""``nn.distillation_loss`` of teachers whose logits, or their quotients by the temperature, are large beside their
distances, on the NumPy backend: only distances count, and keep their digits."""

import numpy as np
import pytest

import openpacho as p
from oracle import blocks
from test_nn_losses import put, within

FLOATS = [np.float32, np.float64]
# (what all of the teacher's logits are moved by, temperature)
OFFSETS = [(30000.0, 1.0), (-30000.0, 0.3), (500.0, 0.01), (7.0, 3.0)]


def check_offsets(backend, vocab, dtype, offset, temperature, rest, rows=6):
    rng = np.random.default_rng(vocab)
    entries = max(1, min(20, vocab // 2))
    z = (temperature * 2 * rng.standard_normal((rows, vocab))).astype(dtype)
    order = np.stack([rng.permutation(vocab)[:entries] for _ in range(rows)])
    listed = (offset + temperature * rng.standard_normal((rows, entries))).astype(dtype)
    others = (listed.max(1).astype(np.longdouble) / np.longdouble(temperature) + rng.standard_normal(rows)).astype(dtype) if rest else None
    listed[1, entries // 2 :] = -np.inf
    if rest:
        others[2], listed[3] = -np.inf, -np.inf
    elif entries < 2:
        listed[1] = 0
    values, units = blocks.distillation_loss(z, order, listed, others, temperature=temperature)
    arrays = put(backend, z, order, listed, others)
    found = p.nn.distillation_loss_grad(*arrays, temperature=temperature)
    for got, want, unit in zip(found, values, units):
        within(got, want, unit, dtype)
    for got, same in zip(p.nn.distillation_loss(*arrays, temperature=temperature), found):
        np.testing.assert_array_equal(p.asnumpy(got), p.asnumpy(same))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rest", [True, False])
@pytest.mark.parametrize("offset,temperature", OFFSETS)
@pytest.mark.parametrize("vocab", [2, 9, 60])
def test_offsets(numpy_backend, vocab, offset, temperature, rest, dtype):
    check_offsets(numpy_backend, vocab, dtype, offset, temperature, rest)
