"""``nn.distillation_loss`` where the student gives the whole rest of the vocabulary less than the type's least
exponential, on the NumPy backend: the rest's logarithm and its gradient are finite all the same."""

import numpy as np
import pytest

import openpacho as p
from oracle import blocks
from test_nn_losses import put, within

FLOATS = [np.float32, np.float64]
GAPS = [60, 80, 87.5, 100, 103.9, 140, 400, 740, 1000, 5000]  # the oracle's exponentials end at 11300
VOCABULARIES = [2, 3, 9, 40, 300]


def far_inputs(vocab, dtype, temperature, gap, rows=7):
    """Rows whose unlisted logits lie `gap` temperatures below the listed ones and further; some rows as others are,
    some with a single unlisted logit nearby, some with forbidden ones among them."""
    rng = np.random.default_rng(vocab)
    entries = max(1, min(6, vocab // 3))
    z = rng.uniform(-1, 1, (rows, vocab))
    order = np.stack([rng.permutation(vocab)[:entries] for _ in range(rows)])
    below = gap + 30 * rng.random((rows, vocab))
    np.put_along_axis(below, order, 0, axis=1)
    below[1] = 0
    if vocab > entries + 1:
        left = np.setdiff1d(np.arange(vocab), order[2])
        below[2, left[len(left) // 2]] = 3
        below[3, np.setdiff1d(np.arange(vocab), order[3])[:-1]] = np.inf
    listed, rest = rng.standard_normal((rows, entries)), rng.standard_normal(rows)
    rest[5] = -np.inf
    return [(temperature * (z - below)).astype(dtype), order, (temperature * listed).astype(dtype), rest.astype(dtype)]


def flushed(given, temperature, dtype):
    """What gradients (rows, 1) lose where exponentials end at the type's least normal number, `tiny`.

    An unlisted logit's is exp((z - m) / T) (1 / S - p_rest / R) / (T count) with R relative to the row's largest
    logit m while it is at least 2^-64 (2^-900), else q - exp((z - m') / T) p_rest / R' with R' >= 1: an exponential that
    is off by tiny makes tiny (1 + p_rest / R), or 2 tiny.
    """
    z, order, listed, rest = (v.astype(np.longdouble) if v.dtype.kind == "f" else v for v in given)
    distance = (z - z.max(1, keepdims=True)) / temperature
    np.put_along_axis(distance, order, -np.inf, axis=1)
    mass = np.exp(distance).sum(1, keepdims=True)
    teacher = np.concatenate([listed / temperature, rest[:, None]], 1)
    p_rest = np.exp(rest[:, None] - teacher.max(1, keepdims=True))
    near = mass > (2.0**-65 if dtype == np.float32 else 2.0**-901)
    return np.finfo(dtype).tiny * np.where(near, 1 + p_rest / np.where(near, mass, 1), 2) / (temperature * len(z))


def check_far_rest(backend, vocab, dtype, gap, temperature=0.5):
    given = far_inputs(vocab, dtype, temperature, gap)
    with np.errstate(invalid="ignore", divide="ignore"):  # of forbidden logits
        values, units = blocks.distillation_loss(*given, temperature=temperature)
        least = flushed(given, temperature, dtype)
    arrays = put(backend, *given)
    found = p.nn.distillation_loss_grad(*arrays, temperature=temperature)
    for got, want, unit, extra in zip(found, values, units, (0, 0, least)):
        assert np.isfinite(want.astype(np.float64)).all()
        within(got, want, np.where(np.isfinite(unit), unit, 0) + extra / (np.finfo(dtype).eps / 2), dtype)
    for got, same in zip(p.nn.distillation_loss(*arrays, temperature=temperature), found):
        np.testing.assert_array_equal(p.asnumpy(got), p.asnumpy(same))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("vocab", VOCABULARIES)
def test_far_rest(numpy_backend, vocab, gap, dtype):
    check_far_rest(numpy_backend, vocab, dtype, gap)


def check_far_rest_by_hand(backend, dtype):
    """One listed logit of 120, two others of 0: p = (e / (1 + e), 1 / (1 + e)), q = (1, 2 exp(-120))."""
    p_list, p_rest = (v.astype(dtype) for v in (np.e / (1 + np.e) * np.ones(1), 1 / (1 + np.e) * np.ones(1)))
    z = np.array([[120, 0, 0], [30000, 0, 0], [1000, 0, -1000]], dtype)
    loss, losses, grad = (p.asnumpy(v) for v in p.nn.distillation_loss_grad(
        *put(backend, z, np.zeros((3, 1), int), np.ones((3, 1), dtype), np.zeros(3, dtype)), count=1))  # fmt: skip
    entropy = p_list * np.log(p_list) + p_rest * np.log(p_rest)
    # A handful of roundings each.
    one = np.finfo(dtype).eps
    want = np.concatenate([entropy + p_rest * (120 - np.log(2)), entropy + p_rest * (30000 - np.log(2)), entropy + p_rest * 1000])
    np.testing.assert_allclose(losses, want, rtol=16 * one)
    np.testing.assert_allclose(loss, want.sum(), rtol=16 * one)
    np.testing.assert_allclose(grad[:2], np.concatenate([p_rest, -p_rest / 2, -p_rest / 2] * 2).reshape(2, 3), rtol=32 * one)
    np.testing.assert_allclose(grad[2], np.concatenate([p_rest, -p_rest, 0 * p_rest]), rtol=32 * one, atol=0)


@pytest.mark.parametrize("dtype", FLOATS)
def test_far_rest_by_hand(numpy_backend, dtype):
    check_far_rest_by_hand(numpy_backend, dtype)


def check_nothing_left(backend, dtype, vocab=5):
    """A rest that the student forbids altogether: infinite where the teacher gives it mass, no matter where it gives none."""
    z = np.full((3, vocab), -np.inf, dtype)
    z[:, 0], z[2, 1] = 3, -5000
    order, listed = np.zeros((3, 1), int), np.zeros((3, 1), dtype)
    rest = np.array([0, -np.inf, -np.inf], dtype)
    loss, losses, grad = (p.asnumpy(v) for v in p.nn.distillation_loss_grad(*put(backend, z, order, listed, rest)))
    assert loss == np.inf and losses[0] == np.inf and not losses[1:].any()
    assert np.isfinite(grad).all() and not grad[1:].any()


@pytest.mark.parametrize("dtype", FLOATS)
def test_nothing_left(numpy_backend, dtype):
    check_nothing_left(numpy_backend, dtype)
