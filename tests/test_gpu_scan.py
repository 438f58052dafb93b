"""The selective scan on the device: against the definition over lengths, channels, groups and states on both sides
of every choice of the kernels, and with values that must not pass a reset or a row's end."""

import numpy as np
import pytest

import openpacho as p
from test_nn_blocks import check_scan, check_scan_goes_on, check_scan_leaves_unread, put_scan, scan_inputs

pytestmark = pytest.mark.gpu

# (batch, time, channels, groups, states): single steps, tiles and one more, one to sixteen waves and states that
# pad them, channels of part of a wave and of several, groups of each; more states than a launch takes.
SIZES = [(1, 1, 1, 1, 1), (2, 1, 4, 2, 3), (2, 7, 6, 2, 4), (1, 20, 3, 1, 16), (3, 5, 4, 4, 2), (2, 16, 65, 1, 16), (1, 17, 130, 2, 8),
         (2, 33, 64, 1, 5), (1, 40, 70, 1, 32), (1, 19, 9, 3, 33), (2, 8, 66, 1, 64), (1, 9, 5, 1, 65), (1, 18, 3, 1, 256), (3, 31, 192, 2, 17),
         (0, 3, 4, 1, 2), (2, 0, 4, 2, 3), (2, 3, 0, 0, 4), (60, 3, 200, 1, 4)]  # fmt: skip


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("full,resets,lengths", [(True, True, True), (False, False, False), (True, False, True), (False, True, False)])
@pytest.mark.parametrize("sizes", SIZES)
def test_scan(hip, sizes, full, resets, lengths, dtype):
    print(sizes, full, resets, lengths, dtype, flush=True)
    check_scan(hip, sizes, dtype, full, resets, lengths)


# Rows in parts: few, many, resets in some parts and rows that end in the first ones.
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("full,resets,lengths", [(True, True, True), (True, False, False), (False, False, True)])
@pytest.mark.parametrize("sizes", [(1, 129, 5, 1, 4), (2, 700, 20, 2, 16), (1, 2100, 3, 1, 3), (5, 200, 70, 1, 20)])
def test_rows_in_parts(hip, sizes, full, resets, lengths, dtype):
    print(sizes, full, resets, lengths, dtype, flush=True)
    check_scan(hip, sizes, dtype, full, resets, lengths, seed=3)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("sizes", [(4, 31, 6, 2, 3), (4, 300, 70, 1, 16), (200, 33, 65, 1, 8)])
def test_scan_leaves_unread(hip, sizes, dtype):
    print(sizes, dtype, flush=True)
    check_scan_leaves_unread(hip, sizes, dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("sizes", [(2, 9, 6, 2, 4), (3, 40, 70, 1, 17)])
def test_scan_goes_on(hip, sizes, dtype):
    check_scan_goes_on(hip, dtype, sizes)


def test_repeated_calls_give_the_same_bits(hip):
    for sizes in ((3, 260, 130, 2, 16), (1, 3000, 64, 1, 8)):
        given, grad, grad_state = scan_inputs(sizes, np.float32, 1)
        arrays, options = put_scan(hip, given)
        grad, grad_state = p.asarray(grad, backend=hip), p.asarray(grad_state, backend=hip)
        calls = [
            (*p.nn.selective_scan(*arrays, **options), *p.nn.selective_scan_grad(grad, *arrays, **options, grad_state=grad_state)) for _ in range(3)
        ]
        for again in calls[1:]:
            for one, two in zip(again, calls[0]):
                np.testing.assert_array_equal(p.asnumpy(one), p.asnumpy(two))
        for name, array in zip(("x", "delta", "a_log", "b", "c", "skip", "gate", "initial"), arrays):
            np.testing.assert_array_equal(p.asnumpy(array), given[name])


def test_the_largest_arrays(hip):
    # Nearly 2^31 elements of x, and steps past 2^32 bytes: the end, from the state before it, has the bits that it has there.
    rows, time, channels, some = 2, 262143, 4095, 96
    rng = p.random.default_rng(2, backend=hip)
    x = rng.normal(0, 1, (rows, time, channels), dtype=np.float32)
    b = rng.normal(0, 1, (rows, time, 1, 2), dtype=np.float32)
    a_log = rng.normal(0, 1, (channels, 2), dtype=np.float32)
    first = p.nn.selective_scan(x[:, : time - some], x[:, : time - some], a_log, b[:, : time - some], b[:, : time - some])[1]
    y, last = p.nn.selective_scan(x, x, a_log, b, b)
    end = slice(time - some, time)
    want, want_last = p.nn.selective_scan(x[:, end], x[:, end], a_log, b[:, end], b[:, end], initial=first)
    # Parts and tiles stand elsewhere: states that forget within some tens of steps agree to their rounding.
    np.testing.assert_allclose(p.asnumpy(y[:, end]), p.asnumpy(want), rtol=0, atol=2e-4)
    np.testing.assert_allclose(p.asnumpy(last), p.asnumpy(want_last), rtol=0, atol=2e-4)
    del y
    found = p.nn.selective_scan_grad(x, x, x, a_log, b, b)
    alone = p.nn.selective_scan_grad(x[:, end], x[:, end], x[:, end], a_log, b[:, end], b[:, end], initial=first)
    for name in ("x", "delta", "b", "c"):
        got, want = p.asnumpy(getattr(found, name)[:, end]), p.asnumpy(getattr(alone, name))
        size = np.abs(want).max()
        np.testing.assert_allclose(got, want, rtol=0, atol=2e-5 * size, err_msg=name)
    del found
    hip.release_cached_memory()


def test_refusals_at_the_library(hip):
    z = p.zeros((4, 8), dtype=np.float32, backend=hip)._data.ptr
    with hip._active():
        for code, index, sizes, pointer in [(1, 2, (1, 2, 4, 1, 2), z), (5, 3, (1, 2, 4, 1, 2), z), (5, 2, (-1, 2, 4, 1, 2), z), (5, 2, (1, 2, 4, 3, 2), z),
                                            (5, 2, (1, 2, 4, 0, 2), z), (5, 2, (1, 2, 4, 1, 0), z), (5, 2, (1, 2, 4, 1, 257), z), (5, 2, (1, 2, 4, 1, 2), None)]:  # fmt: skip
            with pytest.raises(ValueError):
                hip._call("hp_selective_scan", code, index, pointer, *[z] * 4, *[None] * 6, z, z, *sizes)
            with pytest.raises(ValueError):
                hip._call("hp_selective_scan_grad", code, index, pointer, None, *[z] * 5, *[None] * 6, *[z] * 9, *sizes)
