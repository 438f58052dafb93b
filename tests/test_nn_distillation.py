"""``nn.distillation_loss`` on the NumPy backend: values and gradients against the definition and
against differences, lists with gaps and repeats, masks, and what it refuses."""

import numpy as np
import pytest

import openpacho as p
from oracle import blocks
from test_nn_losses import differences, put, within

FLOATS = [np.float32, np.float64]


def inputs(rows, vocab, entries, dtype, seed=0, rest=True, masked=True, index=np.int64, gaps=True):
    rng = np.random.default_rng(seed)
    logits = (3 * rng.standard_normal((rows, vocab))).astype(dtype)
    teacher = logits + 2 * rng.standard_normal((rows, vocab))
    order = np.argsort(-teacher, axis=1)[:, :entries].astype(index)
    listed = np.take_along_axis(teacher, order, 1).astype(dtype)
    others = np.full(rows, -np.inf, dtype)
    if vocab > entries:
        left = np.take_along_axis(teacher, np.argsort(-teacher, axis=1)[:, entries:], 1)
        others = np.log(np.exp(left).sum(1)).astype(dtype)
    if gaps and entries > 1:  # lists that end before the others do, and names in no order
        for row in range(0, rows, 3):
            listed[row, entries // 2 :], order[row, entries // 2 :] = -np.inf, rng.choice([-1, vocab, 2**31 - 1, -(2**31)])
        shuffle = rng.permutation(entries)
        listed, order = listed[:, shuffle], order[:, shuffle]
    mask = rng.random(rows) < 0.7 if masked else None
    if masked:
        out = np.flatnonzero(~mask)
        logits[out[::2]], listed[out], others[out], order[out] = np.nan, np.nan, np.inf, -7
    return logits, order, listed, others if rest else None, mask


def check(backend, rows, vocab, entries, dtype, seed=0, rest=True, masked=True, index=np.int64, **options):
    given = inputs(rows, vocab, entries, dtype, seed, rest, masked, index)
    logits, order, listed, others, mask = put(backend, *given)
    options.setdefault("temperature", 1.5)
    values, units = blocks.distillation_loss(*given, options["temperature"], options.get("count"))
    found = p.nn.distillation_loss_grad(logits, order, listed, others, mask=mask, **options)
    for got, want, unit in zip(found, values, units):
        finite = np.isfinite(want)
        np.testing.assert_array_equal(p.asnumpy(got)[~finite], want[~finite].astype(dtype))
        within(p.asarray(p.asnumpy(got)[finite]), want[finite], unit[finite], dtype)
    if mask is not None:
        out = ~given[4]
        assert not p.asnumpy(found[1])[out].any() and not p.asnumpy(found[2])[out].any()
    for got, same in zip(p.nn.distillation_loss(logits, order, listed, others, mask=mask, **options), found):
        np.testing.assert_array_equal(p.asnumpy(got), p.asnumpy(same))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rest", [True, False])
@pytest.mark.parametrize("rows,vocab,entries", [(1, 1, 1), (1, 2, 1), (9, 5, 4), (40, 33, 8), (5, 300, 64), (7, 20, 20)])
def test_distillation(numpy_backend, rows, vocab, entries, rest, dtype):
    check(numpy_backend, rows, vocab, entries, dtype, seed=rows, rest=rest)
    check(numpy_backend, rows, vocab, entries, dtype, seed=vocab, rest=rest, masked=False, index=np.int32, temperature=1.0, count=7)


def test_gradient_matches_differences(numpy_backend):
    for rest in (True, False):
        logits, order, listed, others, _ = inputs(5, 7, 3, np.float64, 1, rest, False)
        mask = np.array([True, False, True, True, True])
        options = dict(mask=mask, temperature=2.0)
        found = p.nn.distillation_loss_grad(p.asarray(logits), order, listed, others, **options)[2]
        want = differences(lambda z: p.nn.distillation_loss(p.asarray(z), order, listed, others, **options)[0].item(), logits)
        # Central differences: third derivatives of order 1 times step^2, rounding over the step.
        np.testing.assert_allclose(p.asnumpy(found), want, atol=1e-8)


def check_repeats(backend, dtype, vocab=40):
    """An index that stands twice is two entries of the sum, and one name of the list."""
    rng = np.random.default_rng(0)
    z = rng.standard_normal((3, vocab)).astype(dtype)
    order = np.array([[3, 9, 3, 3], [1, 1, 1, 1], [0, 2, 2, vocab - 1]])
    listed = rng.standard_normal((3, 4)).astype(dtype)
    for others in (None, rng.standard_normal(3).astype(dtype)):
        values, units = blocks.distillation_loss(z, order, listed, others)
        found = p.nn.distillation_loss_grad(*put(backend, z, order, listed, others))
        for got, want, unit in zip(found, values, units):
            within(got, want, unit, dtype)


@pytest.mark.parametrize("dtype", FLOATS)
def test_repeats(numpy_backend, dtype):
    check_repeats(numpy_backend, dtype)


def check_edges(backend, dtype):
    inf, low = np.inf, np.finfo(dtype).min
    one = np.finfo(dtype).eps

    def loss(z, order, listed, others=None, **options):
        given = put(backend, np.array(z, dtype), np.array(order), np.array(listed, dtype), None if others is None else np.array(others, dtype))
        found = [p.asnumpy(v) for v in p.nn.distillation_loss_grad(*given, **options)]
        for a, b in zip(found, p.nn.distillation_loss(*given, **options)):
            np.testing.assert_array_equal(a, p.asnumpy(b))
        return found

    # Forbidden logits of the student: an infinite loss where the teacher wants one, and gradient 0 of the others.
    value, each, grad = loss([[0, -inf, 1], [0, -inf, 1]], [[0, 1], [0, 2]], [[0, 0], [0, 0]])
    assert value == inf and each[0] == inf and np.isfinite(each[1]) and np.isfinite(grad).all() and grad[1, 1] == 0
    np.testing.assert_allclose(grad[0, 1], -0.25, rtol=4 * one)  # half of p, over two rows
    # The type's lowest value is a number.
    value, each, grad = loss([[low, 0, 0]], [[1, 2]], [[0, 0]])
    np.testing.assert_allclose(each, 0, atol=8 * one)
    assert grad[0, 0] == 0
    # All forbidden, a NaN, an index outside: a row that is NaN, alone.
    bad = [[-inf] * 3, [0, np.nan, 0], [0, inf, 0], [0, 1, 2], [0, 1, 2], [0, 1, 2]]
    value, each, grad = loss(bad, [[0], [0], [0], [3], [-1], [1]], [[0]] * 6)
    assert np.isnan(value) and np.isnan(each[:5]).all() and np.isfinite(each[5]) and np.isnan(grad[:5]).all() and np.isfinite(grad[5]).all()
    # A teacher without any mass; one whose mass is all in the rest.
    value, each, grad = loss([[0, 1, 2]] * 2, [[0], [-5]], [[-inf], [-inf]], [-inf, 3.0])
    assert np.isnan(each[0]) and np.isnan(grad[0]).all()
    np.testing.assert_allclose(each[1], 0, atol=8 * one)
    np.testing.assert_allclose(grad[1], 0, atol=8 * one)
    # The whole vocabulary listed, with and without a rest: nothing of q is there for it.
    value, each, grad = loss([[0, 1]] * 2, [[0, 1]] * 2, [[0, 1]] * 2, [-inf, 0.0])
    np.testing.assert_allclose(each[0], 0, atol=8 * one)
    assert each[1] == inf and np.isfinite(grad).all()
    # Infinite teachers are no distribution.
    assert np.isnan(loss([[0, 1]], [[0, 1]], [[inf, 0]])[1]).all()
    # Far apart: the temperature scales both sides; nothing overflows.
    value, each, grad = loss([[5000, 0]], [[0, 1]], [[0, 5000]], temperature=100.0)
    np.testing.assert_allclose(value, 50, rtol=8 * one)
    np.testing.assert_allclose(grad, [[0.01, -0.01]], rtol=16 * one)
    # Nothing kept, nothing there.
    z = p.zeros((2, 3), dtype=dtype, backend=backend)
    found = p.nn.distillation_loss_grad(z, [[9], [9]], p.zeros((2, 1), dtype=dtype, backend=backend), mask=[False, False])
    assert found[0].item() == 0 and not p.asnumpy(found[1]).any() and not p.asnumpy(found[2]).any()
    for rows in ((0,), (0, 3), (2, 0)):
        z, t = (p.zeros(rows + (n,), dtype=dtype, backend=backend) for n in (5, 2))
        found = p.nn.distillation_loss_grad(z, np.zeros(rows + (2,), int), t, p.zeros(rows, dtype=dtype, backend=backend))
        assert found[0].item() == 0 and found[1].shape == rows and found[2].shape == rows + (5,)


@pytest.mark.parametrize("dtype", FLOATS)
def test_edges(numpy_backend, dtype):
    check_edges(numpy_backend, dtype)


def test_refusals(numpy_backend):
    f = p.nn.distillation_loss
    z, t, i = p.zeros((2, 5), dtype="float32"), p.zeros((2, 3), dtype="float32"), np.zeros((2, 3), int)
    f(z, i, t)
    for bad in (np.zeros((2, 0), int), np.zeros((2, 1025), int), np.zeros(2, int), np.zeros((3, 3), int)):
        with pytest.raises(ValueError, match="indices"):
            f(z, bad, t)
    for bad in (np.zeros((2, 3)), np.zeros((2, 3), bool)):
        with pytest.raises(p.UnsupportedDtypeError):
            f(z, bad, t)
    with pytest.raises(ValueError, match="teacher_logits"):
        f(z, i, p.zeros((2, 2), dtype="float32"))
    with pytest.raises(ValueError, match="teacher_rest"):
        f(z, i, t, p.zeros((3,), dtype="float32"))
    with pytest.raises(ValueError, match="mask"):
        f(z, i, t, mask=np.zeros((2, 3), bool))
    for bad in (0.0, -1.0, np.nan, np.inf, 1e-39, 1e38):
        with pytest.raises(ValueError, match="temperature"):
            f(z, i, t, temperature=bad)
    for bad in (0, -3.0, np.nan):
        with pytest.raises(ValueError, match="count"):
            f(z, i, t, count=bad)
    with pytest.raises(ValueError, match="none of it empty"):
        f(p.zeros((2, 0), dtype="float32"), i, t)
    with pytest.raises(p.UnsupportedDtypeError):
        f(z, i, p.zeros((2, 3), dtype="float64"))
    with pytest.raises(NotImplementedError, match="not captured"):
        p.compile(lambda z, t: f(z, i, t)[0])(z, t)
