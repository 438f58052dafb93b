"""``nn.selective_scan`` of states that forget at once, on the NumPy backend."""

import numpy as np
import pytest

import openpacho as p
from oracle import blocks
from test_nn_blocks import put, put_scan, scan_inputs, within

FLOATS = [np.float32, np.float64]
# exp(a_log) within the type but not its product with log2 e; past the type; infinite.
RATES = {np.float32: [88.5, 100, np.inf], np.float64: [709.5, 709.7, 800, np.inf]}
SIZES = [(1, 1, 1, 1, 1), (3, 5, 4, 2, 3), (2, 17, 6, 2, 16)]


def check_rates(backend, sizes, dtype, a_log):
    """A state whose decays are all 0 has the bits of one of a smaller rate whose decays are as well."""
    given, grad, grad_state = scan_inputs(sizes, dtype, sum(sizes))
    rng = np.random.default_rng(0)
    at = rng.random(given["a_log"].shape) < 0.5
    at[0, 0] = True
    results = []
    for value in (50, a_log):  # of a step of 1e-4 and more: exp(-5e17) and less
        given["a_log"][at] = value
        arrays, options = put_scan(backend, given)
        results.append([p.asnumpy(v) for v in p.nn.selective_scan(*arrays, **options)])
        grads = put(backend, grad, grad_state)
        found = p.nn.selective_scan_grad(grads[0], *arrays, **options, grad_state=grads[1])
        results[-1] += [p.asnumpy(v) for v in found]
        if value == 50:
            for got, want in zip(results[-1], blocks.selective_scan(**given)):
                within(got, want, dtype)
            for got, want in zip(found, blocks.selective_scan(**given, grad=grad, grad_state=grad_state)):
                within(got, want, dtype)
    for name, want, got in zip(("y", "last", *found._fields), *results):
        assert np.isfinite(want).all(), name
        np.testing.assert_array_equal(got, want, err_msg=name)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("sizes", SIZES)
def test_rates(numpy_backend, sizes, which, dtype):
    check_rates(numpy_backend, sizes, dtype, RATES[dtype][min(which, len(RATES[dtype]) - 1)])


def check_rates_of_tokens(backend, dtype, sizes=(5, 1, 70, 2, 5)):
    given, _, _ = scan_inputs(sizes, dtype, 1, resets=False, lengths=False)
    results = []
    for value in (50, *RATES[dtype]):
        given["a_log"][::2] = value
        at = {k: None if v is None else p.asarray(v[:, 0] if k in ("x", "delta", "b", "c", "gate") else v, backend=backend) for k, v in given.items()}
        found = p.nn.selective_scan_step(
            at["x"], at["delta"], at["a_log"], at["b"], at["c"], at["initial"], at["skip"], at["gate"], delta_bias=at["delta_bias"]
        )
        results.append([p.asnumpy(v) for v in found])
    for other in results[1:]:
        for want, got in zip(results[0], other):
            assert np.isfinite(want).all()
            np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("dtype", FLOATS)
def test_rates_of_tokens(numpy_backend, dtype):
    check_rates_of_tokens(numpy_backend, dtype)


def check_no_rate(backend, dtype):
    """A rate of NaN spoils its own states, and a rate of 0 keeps them."""
    given, _, _ = scan_inputs((2, 3, 4, 1, 3), dtype, 2, resets=False, lengths=False)
    given["a_log"][1, 2], given["a_log"][3] = np.nan, -np.inf
    given["b"][:] = 0
    arrays, options = put_scan(backend, given)
    last = p.asnumpy(p.nn.selective_scan(*arrays, **options)[1])
    assert np.isnan(last[:, 1, 2]).all() and np.isnan(last).sum() == 2
    np.testing.assert_array_equal(last[:, 3], given["initial"][:, 3])


@pytest.mark.parametrize("dtype", FLOATS)
def test_no_rate(numpy_backend, dtype):
    check_no_rate(numpy_backend, dtype)
