"""The causal convolution on the device: against the definition over lengths, channels and taps on both sides of
every choice of the kernels, and with inputs that no step must see."""

import numpy as np
import pytest

import openpacho as p
from test_nn_blocks import check_conv, check_conv_goes_on, check_conv_leaves_unread, conv_inputs
from test_nn_recurrence import put

pytestmark = pytest.mark.gpu

# (batch, time, channels, taps): single steps, rows shorter than the window, ends of runs, vectors that move back.
SIZES = [(1, 1, 1, 1), (2, 1, 5, 4), (3, 2, 4, 8), (2, 9, 6, 3), (1, 17, 3, 8), (2, 8, 7, 2), (2, 7, 2, 5), (3, 16, 8, 4), (2, 65, 13, 6),
         (1, 130, 64, 7), (5, 33, 257, 4), (2, 64, 1, 4), (0, 3, 4, 4), (2, 0, 4, 3), (2, 3, 0, 4), (70, 5, 9, 4), (1, 1000, 2, 3)]  # fmt: skip


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("carried,resets,lengths", [(True, True, True), (False, False, False), (True, False, True), (False, True, False)])
@pytest.mark.parametrize("sizes", SIZES)
def test_conv(hip, sizes, carried, resets, lengths, dtype):
    print(sizes, carried, resets, lengths, dtype, flush=True)
    check_conv(hip, sizes, dtype, carried, resets, lengths)
    check_conv(hip, sizes, dtype, carried, resets, lengths, bias=False, activation=None, index=np.int32)


# Runs of 8 to 64 steps: as many threads as one plan or the next wants.
@pytest.mark.parametrize("sizes", [(2, 1200, 1100, 4), (4, 2100, 515, 3), (3, 70000, 9, 2)])
def test_long_runs(hip, sizes):
    print(sizes, flush=True)
    batch, time, channels, taps = sizes
    x, weight, bias, initial, starts, ends, d = conv_inputs(sizes, np.float32, 1, spoiled=False)
    given = put(hip, x, weight, bias, initial)
    options = dict(resets=put(hip, starts)[0], lengths=put(hip, ends)[0], activation="silu")
    whole = p.nn.causal_conv(*given, **options)
    grads = p.nn.causal_conv_grad(p.asarray(d, backend=hip), *given, **options)
    # Some channels alone, where the plan is another one, have the same bits but for the sums over steps.
    for low, high in ((0, 3), (channels - 5, channels)):
        part = put(hip, *(v[..., low:high].copy() if v is not weight else v[low:high] for v in (x, weight)))
        part += put(hip, bias[low:high], initial[..., low:high].copy())
        for got, want in zip(whole, p.nn.causal_conv(*part, **options)):
            np.testing.assert_array_equal(p.asnumpy(got)[..., low:high], p.asnumpy(want))
        some = p.nn.causal_conv_grad(p.asarray(d[..., low:high].copy(), backend=hip), *part, **options)
        for which in (0, 3):
            np.testing.assert_array_equal(p.asnumpy(grads[which])[..., low:high], p.asnumpy(some[which]))
        for which in (1, 2):
            one, two = p.asnumpy(grads[which])[low:high], p.asnumpy(some[which])
            # Sums of some thousand terms of size 1 in two orders: runs of 64 terms, each 64 roundings of its size.
            np.testing.assert_allclose(one, two, rtol=0, atol=128 * 2.0**-24 * np.sqrt(batch * time) * 4)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("sizes", [(4, 30, 5, 4), (4, 200, 40, 8), (4, 90, 2, 2)])
def test_conv_leaves_unread(hip, sizes, dtype):
    check_conv_leaves_unread(hip, sizes, dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_conv_goes_on(hip, dtype):
    check_conv_goes_on(hip, dtype)


def test_repeated_calls_give_the_same_bits(hip):
    x, weight, bias, initial, starts, ends, d = conv_inputs((3, 1001, 300, 4), np.float32, 1, spoiled=False)
    given = put(hip, d, x, weight, bias, initial)
    calls = [p.nn.causal_conv_grad(*given, resets=starts, lengths=ends, activation="silu") for _ in range(3)]
    for again in calls[1:]:
        for one, two in zip(again, calls[0]):
            np.testing.assert_array_equal(p.asnumpy(one), p.asnumpy(two))


def test_the_largest_arrays(hip):
    # Nearly 2^31 elements: the end has the bits that it has alone.
    rows, time, channels, some = 2, 524287, 2047, 300
    rng = p.random.default_rng(2, backend=hip)
    x = rng.normal(0, 1, (rows, time, channels), dtype=np.float32)
    weight = rng.normal(0, 1, (channels, 4), dtype=np.float32)
    y, last = p.nn.causal_conv(x, weight, activation="silu")
    dx, _, _, _ = p.nn.causal_conv_grad(x, x, weight, activation="silu")
    end = x[1:, time - some :]
    kept, kept_dx = p.asnumpy(y[1:, time - some + 3 :]), p.asnumpy(dx[1:, time - some :])
    del y, dx, x
    want, want_last = p.nn.causal_conv(end, weight, activation="silu")
    np.testing.assert_array_equal(kept, p.asnumpy(want)[:, 3:])
    np.testing.assert_array_equal(p.asnumpy(last[1:]), p.asnumpy(want_last))
    want = p.nn.causal_conv_grad(end, end, weight, activation="silu")[0]
    np.testing.assert_array_equal(kept_dx[:, 3:], p.asnumpy(want)[:, 3:])
    hip.release_cached_memory()


def test_refusals_at_the_library(hip):
    z = p.zeros((4, 8), dtype=np.float32, backend=hip)._data.ptr
    with hip._active():
        for code, index, sizes, pointer in [(1, 2, (1, 2, 4, 2), z), (5, 3, (1, 2, 4, 2), z), (5, 2, (-1, 2, 4, 2), z), (5, 2, (1, 2, 4, 0), z),
                                            (5, 2, (1, 2, 4, 9), z), (5, 2, (1, 2, 4, 2), None)]:  # fmt: skip
            with pytest.raises(ValueError):
                hip._call("hp_causal_conv", code, index, pointer, z, None, None, None, None, z, z, *sizes, 0)
            with pytest.raises(ValueError):
                hip._call("hp_causal_conv_grad", code, index, pointer, z, z, None, None, None, None, z, z, None, None, *sizes, 0)
