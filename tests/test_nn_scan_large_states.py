"""``nn.selective_scan`` of carried states and gradients near the type's ends, on the NumPy backend."""

from unittest import mock

import numpy as np
import pytest

import openpacho as p
from oracle import blocks
from test_nn_blocks import put, put_scan, scan_inputs, within

FLOATS = [np.float32, np.float64]


def ending_at(dtype):
    """Exponentials that end at the type's least normal number: what is below may be 0, so each is off by that number, and
    a state of 2^110 by 2^110 times it in one step, which later steps' decays carry on as they carry the state."""
    least = np.finfo(dtype).tiny / (np.finfo(dtype).eps / 2)
    whole = blocks.exp

    def exp(v):
        found = whole(v)
        return blocks.Number(found.value, found.units + least)

    return mock.patch.object(blocks, "exp", exp)


def check_large_states(backend, sizes, dtype, full=True):
    """Carried states and gradients of 2^110 (2^1000) leave nothing behind where the decays' product is 0."""
    given, grad, grad_state = scan_inputs(sizes, dtype, 5, True, False, False)
    large = dtype(2.0) ** (110 if dtype == np.float32 else 1000)
    given["initial"] *= large
    given["delta"] = np.abs(given["delta"]) + 4  # steps of 1 and more, rates of 0.1 and more
    given["delta_bias"] = given["delta_bias"] / 3
    arrays, options = put_scan(backend, given)
    with np.errstate(under="ignore"), ending_at(dtype):
        for got, want in zip(p.nn.selective_scan(*arrays, **options), blocks.selective_scan(**given)):
            within(got, want, dtype)
        given["initial"] /= large
        arrays, options = put_scan(backend, given)
        grad_state *= large
        given_grads = put(backend, grad, grad_state)
        found = p.nn.selective_scan_grad(given_grads[0], *arrays, **options, grad_state=given_grads[1])
        for name, got, want in zip(found._fields, found, blocks.selective_scan(**given, grad=grad, grad_state=grad_state)):
            try:
                within(got, want, dtype)
            except AssertionError as exc:
                raise AssertionError(f"gradient of {name}: {exc}") from exc


@pytest.mark.parametrize("dtype", FLOATS)
def test_large_states(numpy_backend, dtype):
    check_large_states(numpy_backend, (1, 400, 3, 1, 3), dtype)


def check_infinite_states(backend, sizes, dtype):
    """An infinite state passes every step whose own decay is not 0, and reaches its own channel alone."""
    given, _, _ = scan_inputs(sizes, dtype, 6, True, False, False)
    given["initial"][0, 1, 0], given["initial"][-1, 0, -1] = np.inf, -np.inf
    arrays, options = put_scan(backend, given)
    y, last = (p.asnumpy(v) for v in p.nn.selective_scan(*arrays, **options))
    want = np.zeros(last.shape)
    want[0, 1, 0], want[-1, 0, -1] = 1, -1
    np.testing.assert_array_equal(np.where(np.isinf(last), np.sign(last), 0), want)
    assert not np.isnan(last).any()
    np.testing.assert_array_equal(np.isfinite(y), np.broadcast_to((want == 0).all(-1)[:, None], y.shape))


@pytest.mark.parametrize("dtype", FLOATS)
def test_infinite_states(numpy_backend, dtype):
    check_infinite_states(numpy_backend, (1, 400, 3, 1, 3), dtype)
