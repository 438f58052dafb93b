"""``nn.gated_recurrence`` on the NumPy backend: values against the definition,
gradients against it and against differences, and what it refuses."""

import numpy as np
import pytest

import openpacho as p
from oracle import training

SIZES = [(1, 1, 1, 1), (3, 1, 5, 5), (2, 7, 6, 6), (2, 9, 6, 2), (1, 30, 4, 1), (0, 3, 4, 2), (2, 0, 4, 4), (2, 3, 0, 0)]
# Units of rounding a step: 4 of each gate, 2 products and a sum, and as many again for steps composed in another order.
UNITS = 20


def make(sizes, dtype, seed=0, state=True, resets=True):
    batch, time, channels, gates = sizes
    rng = np.random.default_rng(seed)
    x, d = (rng.standard_normal((batch, time, channels)).astype(dtype) for _ in range(2))
    gate = (2 * rng.standard_normal((batch, time, gates)) + 1).astype(dtype)
    initial = rng.standard_normal((batch, channels)).astype(dtype) if state else None
    starts = rng.random((batch, time)) < 0.15 if resets else None
    return x, gate, initial, starts, d


def put(backend, *values):
    return [None if v is None else p.asarray(v, backend=backend) for v in values]


def near(got, want, size, dtype, units=UNITS):
    bound = units * np.finfo(dtype).eps / 2 * size + np.finfo(dtype).tiny
    error = np.abs(got.astype(training.WIDE) - want)
    assert got.dtype == dtype and got.shape == want.shape
    assert np.all(error <= bound), float(np.max(error / bound))


def check(backend, sizes, dtype, state, resets):
    x, gate, initial, starts, d = make(sizes, dtype, sum(sizes), state, resets)
    xs, gs, first, rs, ds = put(backend, x, gate, initial, starts, d)
    want, size = training.recurrence(x, gate, initial, starts)
    h = p.nn.gated_recurrence(xs, gs, first, resets=rs)
    near(p.asnumpy(h), want, size, dtype)
    states = p.asnumpy(h)
    values, bounds = training.recurrence_grad(d, x, gate, states, initial, starts)
    found = p.nn.gated_recurrence_grad(ds, xs, gs, h, first, resets=rs)
    assert (found[2] is None) == (initial is None)
    for got, want, size in zip(found, values, bounds):
        if got is not None:
            near(p.asnumpy(got), want, size, dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("state,resets", [(True, True), (False, False), (True, False)])
@pytest.mark.parametrize("sizes", SIZES)
def test_values_and_gradients(numpy_backend, sizes, state, resets, dtype):
    check(numpy_backend, sizes, dtype, state, resets)


def agree(got, want, size, dtype):
    """`near` wherever the definition has a number, and its infinities and NaN elsewhere."""
    finite = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(got[np.isinf(want)], want[np.isinf(want)].astype(dtype))
    near(got[finite], want[finite], size[finite], dtype)


def check_infinite_states(backend, sizes, dtype, resets):
    """An infinite state stays so for as long as no reset drops it, over gates whose product leaves the type;
    past a gate of 0, or beside the other infinity, it is NaN. Gradients do so towards the start."""
    batch, time, channels, gates = sizes
    x, gate, initial, starts, d = make(sizes, dtype, 5, True, resets)
    if resets:
        starts[:] = np.random.default_rng(6).random((batch, time)) < 1.5 / time
    width, middle = channels // gates, time // 2
    given, given_d = x.copy(), d.copy()
    initial[:, 0] = np.inf
    for n, channel in enumerate(range(width, channels, width)):  # one of each further head
        at = (n * 37) % time
        given[:, at, channel], given_d[:, at, channel] = (-1) ** n * np.inf, (-1) ** n * np.inf
        if n % 5 == 1:
            gate[:, middle, channel // width] = -np.inf
        if n % 5 == 2:
            given[:, middle, channel], given_d[:, middle, channel] = -given[:, at, channel], -given_d[:, at, channel]
    with np.errstate(invalid="ignore"):
        want, size = training.recurrence(given, gate, initial, starts)
        agree(p.asnumpy(p.nn.gated_recurrence(*put(backend, given, gate, initial), resets=put(backend, starts)[0])), want, size, dtype)
        initial[:, 0] = 1
        h = training.recurrence(x, gate, initial, starts)[0].astype(dtype)
        values, bounds = training.recurrence_grad(given_d, x, gate, h, initial, starts)
    found = p.nn.gated_recurrence_grad(*put(backend, given_d, x, gate, h, initial), resets=put(backend, starts)[0])
    for got, want, size in zip(found, values, bounds):
        agree(p.asnumpy(got), want, size, dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("resets", [True, False])
@pytest.mark.parametrize("sizes", [(1, 1, 3, 3), (2, 40, 12, 12), (2, 300, 12, 4)])
def test_infinite_states(numpy_backend, sizes, resets, dtype):
    check_infinite_states(numpy_backend, sizes, dtype, resets)


def test_gradients_match_differences(numpy_backend):
    x, gate, initial, starts, d = make((2, 6, 4, 2), np.float64, 3)

    def value(x, gate, initial):
        return float((d * p.asnumpy(p.nn.gated_recurrence(*put(numpy_backend, x, gate, initial), resets=p.asarray(starts)))).sum())

    given = [x, gate, initial]
    h = p.nn.gated_recurrence(*put(numpy_backend, *given), resets=p.asarray(starts))
    found = p.nn.gated_recurrence_grad(p.asarray(d), *put(numpy_backend, x, gate), h, p.asarray(initial), resets=p.asarray(starts))
    step = 1e-6
    for which, got in enumerate(found):
        got = p.asnumpy(got)
        for at in np.ndindex(got.shape):
            ends = []
            for sign in (1, -1):
                moved = [v.copy() for v in given]
                moved[which][at] += sign * step
                ends.append(value(*moved))
            # Central differences: third derivatives of order 1 times step^2, rounding of the sum over the step.
            assert abs(got[at] - (ends[0] - ends[1]) / (2 * step)) < 1e-8


def test_a_step_is_one_token_of_the_recurrence(numpy_backend):
    x, gate, initial, _, _ = make((3, 1, 6, 2), np.float32)
    whole = p.asnumpy(p.nn.gated_recurrence(*put(numpy_backend, x, gate, initial)))
    step = p.nn.gated_recurrence_step(*put(numpy_backend, x[:, 0], gate[:, 0], initial))
    np.testing.assert_array_equal(p.asnumpy(step), whole[:, 0])


def test_leading_axes_and_host_values(numpy_backend):
    x, gate, initial, starts, _ = make((6, 5, 4, 4), np.float32)
    flat = p.asnumpy(p.nn.gated_recurrence(*put(numpy_backend, x, gate, initial), resets=p.asarray(starts)))
    shaped = [v.reshape((2, 3) + v.shape[1:]) for v in (x, gate, initial)]
    got = p.nn.gated_recurrence(p.asarray(shaped[0]), shaped[1], shaped[2], resets=starts.reshape(2, 3, 5))
    np.testing.assert_array_equal(p.asnumpy(got), flat.reshape(2, 3, 5, 4))
    alone = p.nn.gated_recurrence(p.asarray(x[0]), p.asarray(gate[0]), p.asarray(initial[0]), resets=starts[0])
    np.testing.assert_array_equal(p.asnumpy(alone), flat[0])


def test_the_first_operand_may_be_a_host_value(numpy_backend):
    x, gate, initial, starts, d = make((2, 5, 4, 2), np.float32)
    want = p.nn.gated_recurrence(*put(numpy_backend, x, gate, initial), resets=starts)
    # Of the arrays' dtype, whatever the host's is.
    for host in (x, x.astype(np.float64), x.tolist()):
        got = p.nn.gated_recurrence(host, p.asarray(gate), initial, resets=p.asarray(starts))
        assert got.dtype == np.float32
        np.testing.assert_array_equal(p.asnumpy(got), p.asnumpy(want))
        grads = p.nn.gated_recurrence_grad(p.asarray(d), host, gate.tolist(), want)
        for one, two in zip(grads[:2], p.nn.gated_recurrence_grad(*put(numpy_backend, d, x, gate), want)):
            np.testing.assert_array_equal(p.asnumpy(one), p.asnumpy(two))
    step = p.nn.gated_recurrence_step(x[:, 0].astype(np.float64), gate[:, 0].tolist(), p.asarray(initial))
    assert step.dtype == np.float32
    # Without any array of floats the first operand gives the dtype; arrays of integers beside it do not.
    assert p.nn.token_log_probs([[1.0, 2.0]], p.asarray([0])).dtype == np.float64
    loss, _ = p.nn.policy_loss(np.zeros((1, 4)), [0], p.zeros((1,), dtype="float32"), [1.0])
    assert loss.dtype == np.float32
    with pytest.raises(p.UnsupportedDtypeError):
        p.nn.token_log_probs([[1, 2]], p.asarray([0]))
    with pytest.raises(p.UnsupportedDtypeError):
        p.nn.gated_recurrence(x, p.zeros((2, 5, 2), dtype="float32"), p.zeros((2, 4), dtype="float64"))


def test_refusals(numpy_backend):
    x, gate = p.zeros((2, 3, 4), dtype="float32"), p.zeros((2, 3, 4), dtype="float32")
    f = p.nn.gated_recurrence
    for bad in (p.zeros((4,), dtype="float32"), p.zeros((2, 3, 6), dtype="float32")):
        with pytest.raises(ValueError):
            f(bad, gate)
    with pytest.raises(ValueError, match="do not divide"):
        f(x, p.zeros((2, 3, 3), dtype="float32"))
    with pytest.raises(ValueError, match="without channels"):
        f(p.zeros((2, 3, 0), dtype="float32"), gate)
    with pytest.raises(ValueError, match="gates"):
        f(x, p.zeros((2, 3, 0), dtype="float32"))
    with pytest.raises(ValueError):
        f(x, p.zeros((2, 4, 4), dtype="float32"))
    with pytest.raises(ValueError, match="initial"):
        f(x, gate, p.zeros((4,), dtype="float32"))
    with pytest.raises(ValueError, match="resets"):
        f(x, gate, resets=np.zeros((2,), bool))
    with pytest.raises(p.UnsupportedDtypeError):
        f(x, gate, resets=p.zeros((2, 3), dtype="int32"))
    with pytest.raises(p.UnsupportedDtypeError):
        f(x, gate, resets=np.zeros((2, 3)))
    with pytest.raises(p.UnsupportedDtypeError):
        f(x, p.zeros((2, 3, 4), dtype="float64"))
    with pytest.raises(p.UnsupportedDtypeError):
        f(p.zeros((2, 3, 4), dtype="int32"), gate)
    with pytest.raises(ValueError, match="grad"):
        p.nn.gated_recurrence_grad(p.zeros((2, 3), dtype="float32"), x, gate, x)
    with pytest.raises(ValueError, match="h must"):
        p.nn.gated_recurrence_grad(x, x, gate, p.zeros((2, 3), dtype="float32"))
    with pytest.raises(ValueError):
        p.nn.gated_recurrence_step(p.zeros((), dtype="float32"), p.zeros((), dtype="float32"), x)
    with pytest.raises(ValueError, match="state"):
        p.nn.gated_recurrence_step(x, gate, p.zeros((2, 3), dtype="float32"))
    with pytest.raises(NotImplementedError, match="not captured"):
        p.compile(lambda x, g: f(x, g))(x, gate)
    with pytest.raises(NotImplementedError, match="not captured"):
        p.fuse(lambda x, g: f(x, g))(x, gate)


# ---- slow gates ------------------------------------------------------------------


def make_slow(sizes, dtype, seed=0, resets=False):
    """Channels that remember some tens to some thousands of steps, a few of them everything, with states that start large
    in every third channel; resets every 3000 steps or so."""
    batch, time, channels, gates = sizes
    rng = np.random.default_rng(seed)
    x, d = (rng.standard_normal((batch, time, channels)).astype(dtype) for _ in range(2))
    gate = (rng.standard_normal((batch, time, gates)) + rng.uniform(4, 10, gates)).astype(dtype)
    if gates > 2:
        gate[:, :, gates // 2] = np.inf
    initial = (rng.standard_normal((batch, channels)) * np.where(np.arange(channels) % 3, 1, 100)).astype(dtype)
    starts = rng.random((batch, time)) < 1 / 3000 if resets else None
    return x, gate, initial, starts, d


def check_slow(backend, sizes, dtype, resets):
    x, gate, initial, starts, d = make_slow(sizes, dtype, sum(sizes), resets)
    xs, gs, first, rs, ds = put(backend, x, gate, initial, starts, d)
    want, size = training.recurrence(x, gate, initial, starts)
    h = p.nn.gated_recurrence(xs, gs, first, resets=rs)
    near(p.asnumpy(h), want, size, dtype)
    values, bounds = training.recurrence_grad(d, x, gate, p.asnumpy(h), initial, starts)
    found = p.nn.gated_recurrence_grad(ds, xs, gs, h, first, resets=rs)
    for got, want, size in zip(found, values, bounds):
        near(p.asnumpy(got), want, size, dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("resets", [False, True])
def test_slow_gates(numpy_backend, resets, dtype):
    check_slow(numpy_backend, (2, 700, 12, 4), dtype, resets)


def mistakes(state, keep, tile, span):
    """What the carried value before each tile would be off by in three mistakes, from the states (time, channels) and gates:
    the second-last tile left out, the state before the block left out, the block's last tile left out of that state.
    Yields (mistake, first step of the tile, error of the value before it)."""
    for first in range(3 * tile, len(state), tile):
        number = first // tile
        inner = number % span
        block = first - inner * tile  # its first step
        if inner >= 2:
            last = keep[first - tile : first].prod(0)
            yield "tile", first, last * (state[first - 2 * tile - 1] - state[first - tile - 1])
        if number >= span:
            since = keep[block:first].prod(0)
            yield "state", first, -since * state[block - 1]
            yield "publish", first, since * (state[block - tile - 1] - state[block - 1])


# Tiles of the device's kernels, forward and backward, in both types, and both lengths of a block.
@pytest.mark.parametrize("dtype,forward,backward", [(np.float32, 128, 64), (np.float64, 64, 32)])
@pytest.mark.parametrize("span,time", [(16, 2200), (64, 17000)])
def test_slow_gates_show_what_tiles_pass_on(span, time, dtype, forward, backward):
    # A tile that got a wrong value from those before it is off by more than test_slow_gates allows, at its first step already.
    x, gate, initial, _, d = make_slow((1, time, 48, 48), dtype, span)
    unit = 20 * np.finfo(dtype).eps / 2
    h, size = training.recurrence(x, gate, initial)
    keep, take = training.sigmoid(gate[0].astype(training.WIDE)), training.sigmoid(-gate[0].astype(training.WIDE))
    seen = set()
    for what, first, off in mistakes(h[0], keep, forward, span):
        seen.add(what)
        # A state that everything before the block has left does not show it in every channel; some do in every tile.
        assert (np.abs(keep[first] * off) > unit * size[0, first]).sum() >= 2, (what, first)
    (dx, _, _), (bound, _, _) = training.recurrence_grad(d, x, gate, h.astype(dtype), initial)
    # The carried gradient m_t = a_t (g_t + m_{t+1}), in the kernels' order, from the last step.
    carried = np.zeros_like(h[0])
    value = np.zeros_like(h[0, 0])
    for t in reversed(range(time)):
        carried[time - 1 - t] = value = keep[t] * (d[0, t] + value)
    for what, first, off in mistakes(carried, keep[::-1], backward, span):
        seen.add(what + " of gradients")
        t = time - 1 - first  # its dx is off by 1 - a times what is carried
        assert (np.abs(take[t] * off) > unit * bound[0, t]).sum() >= 2, (what, first)
    assert len(seen) == 6
