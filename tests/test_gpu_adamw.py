"""``nn.adamw`` on the device: the NumPy backend's tests, lists of more tensors
than one launch takes, and storage that tensors share."""

import numpy as np
import pytest

import openpacho as p
from test_nn_adamw import OPTIONS, SHAPES, bring, check_codes, check_ends, check_first_step, check_resume, check_steps, make, put

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,bits", [(np.float32, None), (np.float64, None), (np.float32, 8)])
def test_steps(hip, dtype, bits):
    check_steps(hip, SHAPES, dtype, bits)
    check_steps(hip, SHAPES, dtype, bits, seed=1, decays=[0.01 * i for i in range(len(SHAPES))])


@pytest.mark.parametrize("dtype,bits", [(np.float32, None), (np.float64, None), (np.float32, 8)])
@pytest.mark.parametrize("tensors", [95, 96, 97, 250])
def test_lists_of_many_tensors(hip, tensors, dtype, bits):
    rng = np.random.default_rng(tensors)
    shapes = [(int(rng.integers(0, 40)), int(rng.integers(1, 60))) for _ in range(tensors)]
    check_steps(hip, shapes, dtype, bits, count=1, decays=[float(d) for d in rng.random(tensors)])


@pytest.mark.parametrize("bits", [None, 8])
def test_tensors_of_many_chunks(hip, bits):
    check_steps(hip, [(1000, 1003), (7,), (513, 2049)], np.float32, bits, count=1)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_first_step(hip, dtype):
    check_first_step(hip, dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_ends_of_the_type(hip, dtype):
    check_ends(hip, dtype)


def test_codes(hip):
    check_codes(hip)


def test_codes_of_many_values(hip):
    # Roots and shares are correctly rounded: as many codes as these agree with the host's to the last one.
    rng = np.random.default_rng(9)
    values = np.exp(rng.uniform(-40, 3, (4000, 1024))).astype(np.float32) * np.exp(rng.uniform(-30, 30, (4000, 1))).astype(np.float32)
    first = np.where(rng.random(values.shape) < 0.5, values, -values).astype(np.float32)
    params = put(hip, [values])
    state = p.nn.adamw_state(params, state_bits=8, first=put(hip, [first]), second=params)
    host = p.get_backend("numpy")
    want = p.nn.adamw_state(put(host, [values]), state_bits=8, first=put(host, [first]), second=put(host, [values]))
    np.testing.assert_array_equal(bring(state.first)[0], bring(want.first)[0])
    np.testing.assert_array_equal(bring(state.second)[0], bring(want.second)[0])


@pytest.mark.parametrize("bits", [None, 8])
def test_resume(hip, bits):
    check_resume(hip, bits)


def test_new_parameters_are_arrays_like_any_other(hip):
    given, grads, _, _ = make([(33, 65), (65,), (65, 7)], np.float32)
    params = put(hip, given)
    new, state = p.nn.adamw(params, put(hip, grads), p.nn.adamw_state(params), **OPTIONS)
    host = bring(new)
    x = np.linspace(-1, 1, 4 * 33).reshape(4, 33).astype(np.float32)
    wide = [a.astype(np.float64) for a in host]
    net = lambda x, a, b, c: np.tanh(x @ a + b) @ c  # noqa: E731
    want = np.tanh(x @ wide[0] + wide[1]) @ wide[2]
    for f in (net, p.compile(net)):
        np.testing.assert_allclose(p.asnumpy(f(p.asarray(x, backend=hip), *new)), want, rtol=1e-4, atol=1e-5)
    # One of them keeps their block when the others are gone; views and copies hold its values.
    kept = new[1]
    moment = state.first[2]
    values = p.asnumpy(moment)
    del new, state, params
    junk = [p.full((65, 65), 7, dtype=np.float32, backend=hip) for _ in range(8)]
    np.testing.assert_array_equal(p.asnumpy(kept.reshape(5, 13)).ravel(), host[1])
    np.testing.assert_array_equal(p.asnumpy(kept[3:60:2]), host[1][3:60:2])
    np.testing.assert_array_equal(p.asnumpy(moment), values)
    assert len(junk) == 8


def test_a_closed_backend_releases_shared_storage():
    from openpacho._hip import HIPBackend

    own = HIPBackend()
    params = [p.ones((5,), dtype=np.float32, backend=own), p.ones((300,), dtype=np.float32, backend=own)]
    new, state = p.nn.adamw(params, params, p.nn.adamw_state(params, state_bits=8))
    moments = state.first
    own.close()
    for array in (*new, *moments):
        with pytest.raises(RuntimeError):
            p.asnumpy(array)
    with pytest.raises(RuntimeError):
        p.nn.adamw(new, new, state)


def test_memory_returns_to_the_pool(hip):
    hip.synchronize()
    params = [p.ones((700, 700), dtype=np.float32, backend=hip)]
    state = p.nn.adamw_state(params)
    before = hip.pool_stats()["live_bytes"]
    for _ in range(5):
        params, state = p.nn.adamw(params, params, state)
    # The first state and parameters are gone: as many bytes live as before, but for the size classes of the new ones.
    assert hip.pool_stats()["live_bytes"] <= before + (2 << 20)


def test_refusals_at_the_library(hip):
    import ctypes

    a = p.zeros((4,), dtype=np.float32, backend=hip)._data.ptr
    one, sizes, decays = (ctypes.c_void_p * 1)(a), (ctypes.c_int64 * 1)(4), (ctypes.c_double * 1)(0)
    none, below = (ctypes.c_void_p * 1)(None), (ctypes.c_int64 * 1)(-1)
    tail = (0.9, 0.999, 1e-3, 1.0, 1e-8)
    with hip._active():
        for code, bits, count, p_, s_ in [(1, 0, 1, one, sizes), (6, 8, 1, one, sizes), (5, 4, 1, one, sizes), (5, 0, -1, one, sizes),
                                          (5, 0, 1, none, sizes), (5, 0, 1, one, below)]:  # fmt: skip
            with pytest.raises(ValueError):
                hip._call("hp_adamw_step", code, bits, count, p_, one, s_, decays, a, a + 4096, a, *tail)
        with pytest.raises(ValueError, match="own"):
            hip._call("hp_adamw_step", 5, 0, 1, one, one, sizes, decays, a, a, a, *tail)
        with pytest.raises(ValueError):
            hip._call("hp_adamw_values", 100, a, 0, a)
        with pytest.raises(ValueError):
            hip._call("hp_adamw_values", 1024, a, 2, a)
