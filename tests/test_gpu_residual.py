"""The residual stream and its norms on the device: against the definition over row lengths and numbers on
both sides of every choice of the kernels, with gates that tokens, sequences and all rows share."""

import numpy as np
import pytest

import openpacho as p
from test_nn_blocks import GATES, check_norm, check_norm_of_no_rows, norm_inputs, put

pytestmark = pytest.mark.gpu

# Rows of part of a team, of whole teams and one more, up to rows that no team holds.
SIZES = [((), 1), ((3,), 3), ((5,), 4), ((2, 9), 5), ((7,), 8), ((130,), 63), ((3, 5), 64), ((2, 5), 65), ((9,), 256), ((5,), 257), ((2, 3), 511),
         ((3,), 513), ((2, 2), 1023), ((3,), 1025), ((5,), 2048), ((2, 2), 2049), ((3,), 4097), ((3,), 8191), ((2, 2), 8193), ((2,), 16385)]  # fmt: skip


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate", list(GATES))
@pytest.mark.parametrize("lead,channels", SIZES)
def test_norm(hip, lead, channels, gate, post, dtype):
    print(lead, channels, gate, post, dtype, flush=True)
    check_norm(hip, lead, channels, dtype, gate, post)


# Workers of several rows, groups within a worker and across some of them, the last ones partly filled.
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("lead,channels", [((3, 701), 40), ((701, 3), 40), ((7, 151), 260), ((4001,), 20), ((2, 301), 1100), ((3, 91), 4200), ((5, 53), 8200), ((40, 260), 3)])
@pytest.mark.parametrize("gate", list(GATES))
def test_many_rows(hip, lead, channels, gate, dtype):
    print(lead, channels, gate, dtype, flush=True)
    check_norm(hip, lead, channels, dtype, gate, True)


@pytest.mark.parametrize("gate", list(GATES))
@pytest.mark.parametrize("lead", [(0,), (0, 3), (3, 0)])
def test_norm_of_no_rows(hip, lead, gate):
    check_norm_of_no_rows(hip, lead, gate)


@pytest.mark.parametrize("channels", [1, 7, 300, 2048, 9001])
def test_rows_stand_alone(hip, channels):
    # A row that is NaN, one that is infinite and one of zeros leave the others as they are.
    lead = (50,)
    x, residual, weight, post, gate, ds, dn = norm_inputs(lead, channels, np.float32, 0, "token", True)
    bad_x, bad_residual = x.copy(), residual.copy()
    bad_x[3, 0], bad_residual[11, -1], bad_x[20], bad_residual[21] = np.nan, np.inf, 0, 0
    rows = [r for r in range(50) if r not in (3, 11, 20, 21)]
    results = []
    for a, b in ((x, residual), (bad_x, bad_residual)):
        arrays = put(hip, a, b, weight)
        options = dict(zip(("post_weight", "gate"), put(hip, post, gate)))
        stream, normed = p.nn.residual_norm(*arrays, **options)
        grads = p.nn.residual_norm_grad(*put(hip, ds, dn), arrays[0], stream, arrays[2], **options)
        results.append([p.asnumpy(v) for v in (stream, normed, grads[0], grads[1], grads[4])])
    for one, two in zip(*results):
        np.testing.assert_array_equal(one[rows], two[rows])
        assert np.isfinite(two[20:22]).all()
    assert np.isnan(results[1][1][3]).all() and np.isnan(results[1][1][11, -1])
    np.testing.assert_array_equal(results[1][0][20], residual[20])


def test_repeated_calls_give_the_same_bits(hip):
    for gate in GATES:
        x, residual, weight, post, gates, ds, dn = put(hip, *norm_inputs((3, 1001), 700, np.float32, 1, gate, True))
        options = dict(post_weight=post, gate=gates)
        stream = p.nn.residual_norm(x, residual, weight, **options)[0]
        calls = [p.nn.residual_norm_grad(ds, dn, x, stream, weight, **options) for _ in range(3)]
        for again in calls[1:]:
            for one, two in zip(again, calls[0]):
                if one is not None:
                    np.testing.assert_array_equal(p.asnumpy(one), p.asnumpy(two))


def test_the_largest_arrays(hip):
    # Nearly 2^31 elements: the last rows have the bits that they have alone.
    rows, channels, some = 1048000, 2047, 60
    rng = p.random.default_rng(2, backend=hip)
    x = rng.normal(0, 1, (rows, channels), dtype=np.float32)
    weight = rng.normal(0, 1, (channels,), dtype=np.float32)
    stream, normed = p.nn.residual_norm(x, x, weight, post_weight=weight)
    last = x[rows - some :]
    want = p.nn.residual_norm(last, last, weight, post_weight=weight)
    for got, value in zip((stream, normed), want):
        np.testing.assert_array_equal(p.asnumpy(got[rows - some :]), p.asnumpy(value))
    del normed
    found = p.nn.residual_norm_grad(x, x, x, stream, weight, post_weight=weight)
    alone = p.nn.residual_norm_grad(last, last, last, want[0], weight, post_weight=weight)
    for got, value in zip(found[:2], alone[:2]):
        np.testing.assert_array_equal(p.asnumpy(got[rows - some :]), p.asnumpy(value))
    del found
    hip.release_cached_memory()


def test_refusals_at_the_library(hip):
    z = p.zeros((4, 8), dtype=np.float32, backend=hip)._data.ptr
    with hip._active():
        for code, rows, channels, divide, scale, eps, pointer in [
            (1, 2, 4, 1, 1.0, 1e-6, z), (5, -1, 4, 1, 1.0, 1e-6, z), (5, 2, 0, 1, 1.0, 1e-6, z), (5, 2, 4, 0, 1.0, 1e-6, z), (5, 3, 4, 2, 1.0, 1e-6, z),
            (5, 2, 4, 1, float("inf"), 1e-6, z), (5, 2, 4, 1, 1.0, 0.0, z), (5, 2, 4, 1, 1.0, float("nan"), z), (5, 2, 4, 1, 1.0, 1e-6, None)]:  # fmt: skip
            with pytest.raises(ValueError):
                hip._call("hp_residual_norm", code, pointer, *[z] * 6, rows, channels, divide, scale, eps)
            with pytest.raises(ValueError):
                hip._call("hp_residual_norm_grad", code, pointer, *[z] * 11, rows, channels, divide, 2, scale, eps)
        with pytest.raises(ValueError, match="gates"):
            hip._call("hp_residual_norm_grad", 5, *[z] * 12, 4, 2, 2, 3, 1.0, 1e-6)
