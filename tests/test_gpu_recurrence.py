"""The gated recurrence on the device: against the definition over lengths,
widths of heads and row numbers on both sides of every choice of the kernels,
and with values that must not pass a reset."""

import numpy as np
import pytest

import openpacho as p
from oracle import training
from test_nn_recurrence import check, make, near, put

pytestmark = pytest.mark.gpu

# (rows, time, channels, gates): one step, partial and several runs of waves, partial and several
# groups of 64 channels; heads of 3, 64, 66, 100, 125 and 128 channels: packed, whole and in pieces.
SIZES = [
    (1, 1, 1, 1), (3, 1, 65, 65), (5, 2, 13, 13), (2, 17, 64, 64), (1, 1000, 3, 3), (2, 129, 70, 70), (4, 257, 130, 130),
    (33, 65, 2, 2), (2, 33, 12, 4), (3, 5, 64, 1), (2, 9, 66, 1), (1, 515, 200, 2), (2, 130, 125, 1), (2, 40, 256, 2),
    (1, 300, 96, 96), (7, 31, 40, 8), (0, 3, 4, 2), (2, 0, 4, 4), (2, 3, 0, 0),
    # the ends of runs, of workgroups and of two of them, and tiles beyond
    (2, 4, 5, 5), (2, 5, 5, 1), (1, 8, 70, 70), (1, 16, 70, 35), (1, 32, 9, 9), (1, 63, 9, 3), (1, 64, 66, 66), (1, 128, 9, 1),
    (1, 192, 65, 65), (1, 193, 6, 6), (1, 256, 6, 2), (1, 384, 3, 3), (1, 385, 3, 1), (1, 513, 130, 1),
]  # fmt: skip


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("state,resets", [(True, True), (False, False), (True, False)])
@pytest.mark.parametrize("sizes", SIZES)
def test_values_and_gradients(hip, sizes, state, resets, dtype):
    print(sizes, state, resets, dtype, flush=True)
    check(hip, sizes, dtype, state, resets)


# Several blocks of tiles, of 16 (from 32 groups of channels on) and of 64.
@pytest.mark.parametrize("sizes", [(1, 20000, 5, 5), (1, 5001, 130, 2), (2, 4099, 65, 65), (1, 2100, 1030, 1030), (3, 2049, 400, 4),
                                   (2, 2100, 1030, 1030), (1, 2200, 2050, 1)])  # fmt: skip
def test_long_rows(hip, sizes):
    print(sizes, flush=True)
    check(hip, sizes, np.float32, True, True)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_a_reset_drops_whatever_was_before(hip, dtype):
    x, gate, initial, starts, d = make((2, 300, 66, 66), dtype)
    at = 150
    starts[:, at] = True
    bad, bad_d = x.copy(), d.copy()
    bad[0, :at], bad[1, at - 1] = np.nan, np.inf
    bad_d[:, at:] = np.inf
    xs, gs, first, rs, ds = put(hip, bad, gate, initial, starts, bad_d)
    h = p.nn.gated_recurrence(xs, gs, first, resets=rs)
    want, size = training.recurrence(x, gate, initial, starts)
    near(p.asnumpy(h)[:, at:], want[:, at:], size[:, at:], dtype)
    assert np.isnan(p.asnumpy(h)[0, at - 1]).all()
    # The gradient of what is after the reset does not reach what is before it.
    clean = training.recurrence(x, gate, initial, starts)[0].astype(dtype)
    d0 = d.copy()
    d0[:, at:] = 0
    values, bounds = training.recurrence_grad(d0, x, gate, clean, initial, starts)
    found = p.nn.gated_recurrence_grad(ds, *put(hip, x, gate, clean, initial), resets=rs)
    for got, want, size in zip(found[:2], values, bounds):
        near(p.asnumpy(got)[:, :at], want[:, :at], size[:, :at], dtype)
    near(p.asnumpy(found[2]), values[2], bounds[2], dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_gates_at_their_ends(hip, dtype):
    # Shut and open gates, and gates whose sigmoid is near 0 or 1: exact, or to full relative precision.
    gate = np.array([np.inf, -np.inf, 80.0, -80.0, 30.0, -30.0, 0.0, 1e-4], dtype)
    x = np.linspace(1, 2, 8).astype(dtype)
    first = np.linspace(-3, -1, 8).astype(dtype)
    h = p.asnumpy(p.nn.gated_recurrence(*put(hip, x[None], gate[None], first)))[0]
    assert h[0] == first[0] and h[1] == x[1]
    want, size = training.recurrence(x[None, None], gate[None, None], first[None])
    near(h, want[0, 0], size[0, 0], dtype)
    # dx is the gradient times 1 - sigmoid: small values keep their digits.
    one = np.ones((1, 8), dtype)
    dx = p.asnumpy(p.nn.gated_recurrence_grad(*put(hip, one, x[None], gate[None], h[None], first))[0])[0]
    with np.errstate(over="ignore"):
        want = training.sigmoid(-gate.astype(training.WIDE))
    near(dx, want, want, dtype)


@pytest.mark.parametrize("sizes,dtype", [((9, 4100, 2048, 2048), np.float32), ((9, 4100, 2048, 4), np.float32), ((9, 4100, 2048, 256), np.float32),
                                         ((4100, 20, 1024, 1024), np.float32), ((9, 2100, 2048, 2048), np.float64)])  # fmt: skip
def test_more_states_than_the_last_cache_holds(hip, sizes, dtype):
    # They are stored past it; fewer rows of the same are not, and have the same bits.
    print(sizes, dtype, flush=True)
    rows, time, channels, gates = sizes
    rng = p.random.default_rng(1, backend=hip)
    x, gate = rng.normal(0, 1, (rows, time, channels), dtype=dtype), rng.normal(2, 1, (rows, time, gates), dtype=dtype)
    resets = np.random.default_rng(1).random((rows, time)) < 0.01
    h = p.nn.gated_recurrence(x, gate, resets=resets)
    for part in (slice(0, 2), slice(rows - 2, rows)):
        fewer = p.nn.gated_recurrence(x[part], gate[part], resets=resets[part])
        np.testing.assert_array_equal(p.asnumpy(h[part]), p.asnumpy(fewer))


def test_repeated_calls_give_the_same_bits(hip):
    x, gate, initial, starts, d = make((2, 700, 250, 2), np.float32)
    given = put(hip, x, gate, initial, starts, d)
    xs, gs, first, rs, ds = given
    h = p.nn.gated_recurrence(xs, gs, first, resets=rs)
    grads = p.nn.gated_recurrence_grad(ds, xs, gs, h, first, resets=rs)
    for _ in range(3):
        np.testing.assert_array_equal(p.asnumpy(p.nn.gated_recurrence(xs, gs, first, resets=rs)), p.asnumpy(h))
        for one, two in zip(p.nn.gated_recurrence_grad(ds, xs, gs, h, first, resets=rs), grads):
            np.testing.assert_array_equal(p.asnumpy(one), p.asnumpy(two))
    for before, array in zip((x, gate, initial, starts, d), given):
        np.testing.assert_array_equal(p.asnumpy(array), before)


def test_refusals_at_the_library(hip):
    x = p.zeros((1, 2, 4), dtype=np.float32, backend=hip)
    with hip._active():
        for sizes, code, pointer in [((1, 2, 4, 3), 5, x._data.ptr), ((1, 2, 4, 0), 5, x._data.ptr), ((-1, 2, 4, 4), 5, x._data.ptr),
                                     ((1, 2, 4, 4), 1, x._data.ptr), ((1, 2, 4, 4), 5, None)]:  # fmt: skip
            with pytest.raises(ValueError):
                hip._call("hp_gated_recurrence", code, pointer, x._data.ptr, None, None, x._data.ptr, *sizes)
            with pytest.raises(ValueError):
                hip._call("hp_gated_recurrence_grad", code, pointer, *[x._data.ptr] * 3, None, None, *[x._data.ptr] * 2, None, *sizes)
