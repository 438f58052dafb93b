"""The convolution, the selective scan and the residual norms of ``nn`` on the NumPy backend: values and
gradients against the definitions and against differences, what they leave unread, and what they refuse."""

import numpy as np
import pytest

import openpacho as p
from oracle import blocks
from test_nn_recurrence import put

FLOATS = [np.float32, np.float64]


def within(got, want, dtype):
    got = p.asnumpy(got)
    assert got.dtype == dtype and got.shape == want.value.shape
    error = np.abs(got.astype(blocks.WIDE) - want.value)
    bound = np.finfo(dtype).eps / 2 * want.units + np.finfo(dtype).tiny
    assert np.all(error <= bound), float(np.max(error / bound))


# ---- causal convolution ----------------------------------------------------------


def conv_inputs(sizes, dtype, seed=0, carried=True, resets=True, lengths=True, spoiled=True):
    """`spoiled`: what must not count is NaN or infinite."""
    batch, time, channels, taps = sizes
    rng = np.random.default_rng(seed)
    x, d = (rng.standard_normal((batch, time, channels)).astype(dtype) for _ in range(2))
    weight, bias = rng.standard_normal((channels, taps)).astype(dtype), rng.standard_normal(channels).astype(dtype)
    initial = rng.standard_normal((batch, taps - 1, channels)).astype(dtype) if carried else None
    starts = rng.random((batch, time)) < 0.15 if resets else None
    ends = rng.integers(-1, time + 2, batch) if lengths else None
    if lengths and spoiled:
        for row, end in enumerate(ends):
            x[row, max(0, end) :], d[row, max(0, end) :] = np.nan, np.inf
    if resets and spoiled and time > 3:
        # In the first row every step up to the middle is followed by a reset.
        starts[0, time // 2] = True
        x[0, : time // 2] = np.inf
        d[0, : time // 2] = 0
        if carried:
            initial[0] = np.nan
    return x, weight, bias, initial, starts, ends, d


def check_conv(backend, sizes, dtype, carried=True, resets=True, lengths=True, bias=True, activation="silu", index=np.int64):
    x, weight, b, initial, starts, ends, d = conv_inputs(sizes, dtype, sum(sizes), carried, resets, lengths, False)
    if not bias:
        b = None
    if ends is not None:
        ends = ends.astype(index)
    xs, ws, bs, first, rs, es, ds = put(backend, x, weight, b, initial, starts, ends, d)
    y, last = p.nn.causal_conv(xs, ws, bs, first, resets=rs, lengths=es, activation=activation)
    want, window = blocks.causal_conv(x, weight, b, initial, starts, ends, activation)
    within(y, want, dtype)
    np.testing.assert_array_equal(p.asnumpy(last), window.astype(dtype))
    found = p.nn.causal_conv_grad(ds, xs, ws, bs, first, resets=rs, lengths=es, activation=activation)
    values = blocks.causal_conv(x, weight, b, initial, starts, ends, activation, grad=d)
    assert (found[2] is None) == (b is None) and (found[3] is None) == (initial is None)
    for got, want in zip(found, values):
        if got is not None:
            within(got, want, dtype)


def check_conv_leaves_unread(backend, sizes, dtype):
    """Inputs behind a row's end and before its reset may be anything where no kept step sees them."""
    clean, spoiled = (conv_inputs(sizes, dtype, 3, spoiled=s) for s in (False, True))
    time = sizes[1]
    middle, ends = time // 2, np.clip(clean[5], 0, time)
    for give in (clean, spoiled):
        give[4][0, middle] = True
        give[6][0, :middle] = 0
    results = []
    for x, weight, bias, initial, starts, lengths, d in (clean, spoiled):
        given = put(backend, x, weight, bias, initial)
        options = dict(resets=p.asarray(starts, backend=backend), lengths=p.asarray(lengths, backend=backend), activation="silu")
        results.append([p.asnumpy(v) for v in p.nn.causal_conv(*given, **options)])
        results[-1] += [p.asnumpy(p.nn.causal_conv_grad(p.asarray(d, backend=backend), *given, **options)[0])]
    one, two = results
    rows = np.arange(sizes[0]) > 0
    np.testing.assert_array_equal(one[0][rows], two[0][rows])
    np.testing.assert_array_equal(one[0][0, middle:], two[0][0, middle:])
    np.testing.assert_array_equal(one[1][rows], two[1][rows])
    if ends[0] >= middle + sizes[3]:
        np.testing.assert_array_equal(one[1][0], two[1][0])
    np.testing.assert_array_equal(one[2][rows], two[2][rows])
    for row, end in enumerate(ends):
        assert not two[0][row, end:].any() and not two[2][row, end:].any()


CONV_SIZES = [(1, 1, 1, 1), (2, 1, 5, 4), (3, 2, 4, 4), (2, 9, 6, 3), (1, 17, 3, 8), (2, 8, 7, 2), (0, 3, 4, 4), (2, 0, 4, 3), (2, 3, 0, 4)]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("carried,resets,lengths", [(True, True, True), (False, False, False), (True, False, True), (False, True, False)])
@pytest.mark.parametrize("sizes", CONV_SIZES)
def test_conv(numpy_backend, sizes, carried, resets, lengths, dtype):
    check_conv(numpy_backend, sizes, dtype, carried, resets, lengths)
    check_conv(numpy_backend, sizes, dtype, carried, resets, lengths, bias=False, activation=None, index=np.int32)


@pytest.mark.parametrize("dtype", FLOATS)
def test_conv_leaves_unread(numpy_backend, dtype):
    check_conv_leaves_unread(numpy_backend, (4, 30, 5, 4), dtype)


def check_conv_goes_on(backend, dtype):
    """Calls that go on from the last inputs, by sequences and by single tokens, have the bits of one call."""
    x, weight, bias, initial, starts, _, _ = conv_inputs((2, 12, 5, 4), dtype, 1, spoiled=False)
    xs, ws, bs, first = put(backend, x, weight, bias, initial)
    whole, end = p.nn.causal_conv(xs, ws, bs, first, resets=p.asarray(starts, backend=backend), activation="silu")
    state, parts = first, []
    for low, high in ((0, 1), (1, 3), (3, 10), (10, 12)):
        y, state = p.nn.causal_conv(xs[:, low:high], ws, bs, state, resets=starts[:, low:high], activation="silu")
        parts.append(p.asnumpy(y))
    np.testing.assert_array_equal(np.concatenate(parts, 1), p.asnumpy(whole))
    np.testing.assert_array_equal(p.asnumpy(state), p.asnumpy(end))
    whole, end = p.nn.causal_conv(xs, ws, bs, first)
    state = first
    for t in range(12):
        y, state = p.nn.causal_conv_step(xs[:, t], ws, state, bs)
        np.testing.assert_array_equal(p.asnumpy(y), p.asnumpy(whole)[:, t])
    np.testing.assert_array_equal(p.asnumpy(state), p.asnumpy(end))


@pytest.mark.parametrize("dtype", FLOATS)
def test_conv_goes_on(numpy_backend, dtype):
    check_conv_goes_on(numpy_backend, dtype)


def differences(value, given, which, step=1e-6):
    found = np.empty_like(given[which])
    for at in np.ndindex(found.shape):
        ends = []
        for sign in (1, -1):
            moved = [None if v is None else v.copy() for v in given]
            moved[which][at] += sign * step
            ends.append(value(moved))
        found[at] = (ends[0] - ends[1]) / (2 * step)
    return found


def test_conv_gradients_match_differences(numpy_backend):
    x, weight, bias, initial, starts, ends, d = conv_inputs((2, 6, 3, 3), np.float64, 2, spoiled=False)
    options = dict(resets=starts, lengths=np.array([6, 4]), activation="silu")

    def value(given):
        return float((d * p.asnumpy(p.nn.causal_conv(*put(numpy_backend, *given), **options)[0])).sum())

    given = [x, weight, bias, initial]
    found = p.nn.causal_conv_grad(p.asarray(d), *put(numpy_backend, *given), **options)
    for which, got in enumerate(found):
        # Central differences: third derivatives of order 10 times step^2, rounding over the step.
        np.testing.assert_allclose(p.asnumpy(got), differences(value, given, which), atol=1e-8)


def test_conv_refusals(numpy_backend):
    f = p.nn.causal_conv
    x, w = p.zeros((2, 3, 4), dtype="float32"), p.zeros((4, 3), dtype="float32")
    for bad in ((4,), (3, 3), (4, 0), (4, 9), (4, 3, 1)):
        with pytest.raises(ValueError, match="weight"):
            f(x, p.zeros(bad, dtype="float32"))
    with pytest.raises(ValueError, match="axes"):
        f(p.zeros((4,), dtype="float32"), w)
    with pytest.raises(ValueError, match="bias"):
        f(x, w, p.zeros((3,), dtype="float32"))
    with pytest.raises(ValueError, match="initial"):
        f(x, w, None, p.zeros((2, 3, 4), dtype="float32"))
    with pytest.raises(ValueError, match="resets"):
        f(x, w, resets=np.zeros((2, 4), bool))
    with pytest.raises(ValueError, match="lengths"):
        f(x, w, lengths=np.zeros(3, int))
    for bad in (np.zeros(2), np.zeros(2, bool)):
        with pytest.raises(p.UnsupportedDtypeError):
            f(x, w, lengths=bad)
    with pytest.raises(ValueError, match="activation"):
        f(x, w, activation="relu")
    with pytest.raises(p.UnsupportedDtypeError):
        f(x, p.zeros((4, 3), dtype="float64"))
    with pytest.raises(p.UnsupportedDtypeError):
        f(p.zeros((2, 3, 4), dtype="int32"), w)
    with pytest.raises(ValueError, match="grad"):
        p.nn.causal_conv_grad(p.zeros((2, 3), dtype="float32"), x, w)
    with pytest.raises(ValueError, match="state"):
        p.nn.causal_conv_step(x[:, 0], w, p.zeros((2, 3, 4), dtype="float32"))
    with pytest.raises(ValueError):
        p.nn.causal_conv_step(p.zeros((), dtype="float32"), w, x)
    with pytest.raises(NotImplementedError, match="not captured"):
        p.compile(lambda x, w: f(x, w)[0])(x, w)


# ---- selective scan ----------------------------------------------------------------

SCAN_NAMES = ("x", "delta", "a_log", "b", "c", "skip", "gate", "initial", "delta_bias", "resets", "lengths")


def scan_inputs(sizes, dtype, seed=0, full=True, resets=True, lengths=True):
    """`full`: with skip, gate, states and bias."""
    batch, time, channels, groups, states = sizes
    rng = np.random.default_rng(seed)

    def normal(*shape):
        return rng.standard_normal(shape).astype(dtype)

    given = {
        "x": normal(batch, time, channels),
        "delta": normal(batch, time, channels),
        "a_log": (0.5 * normal(channels, states)).astype(dtype) + np.log(np.arange(1, states + 1)).astype(dtype) * dtype(0.5),
        "b": normal(batch, time, groups, states),
        "c": normal(batch, time, groups, states),
        "skip": normal(channels) if full else None,
        "gate": normal(batch, time, channels) if full else None,
        "initial": normal(batch, channels, states) if full else None,
        "delta_bias": rng.uniform(-6, 0, channels).astype(dtype) if full else None,
        "resets": rng.random((batch, time)) < 0.1 if resets else None,
        "lengths": rng.integers(-1, time + 2, batch) if lengths else None,
    }
    return given, normal(batch, time, channels), normal(batch, channels, states)


def put_scan(backend, given):
    found = {k: None if v is None else p.asarray(v, backend=backend) for k, v in given.items()}
    return [found[k] for k in SCAN_NAMES[:8]], {k: found[k] for k in SCAN_NAMES[8:]}


def check_scan(backend, sizes, dtype, full=True, resets=True, lengths=True, seed=None):
    given, grad, grad_state = scan_inputs(sizes, dtype, sum(sizes) if seed is None else seed, full, resets, lengths)
    arrays, options = put_scan(backend, given)
    for got, want in zip(p.nn.selective_scan(*arrays, **options), blocks.selective_scan(**given)):
        within(got, want, dtype)
    last = grad_state if full else None
    want = blocks.selective_scan(**given, grad=grad, grad_state=last)
    given_grads = put(backend, grad, last)
    found = p.nn.selective_scan_grad(given_grads[0], *arrays, **options, grad_state=given_grads[1])
    names = ("x", "delta", "a_log", "b", "c", "skip", "gate", "delta_bias", "initial")
    assert found._fields == names
    for name, got, value in zip(names, found, want):
        assert (got is None) == (given[name] is None), name
        if got is not None:
            try:
                within(got, value, dtype)
            except AssertionError as exc:
                raise AssertionError(f"gradient of {name}: {exc}") from exc


SCAN_SIZES = [(1, 1, 1, 1, 1), (2, 1, 4, 2, 3), (2, 7, 6, 2, 4), (1, 20, 3, 1, 16), (3, 5, 4, 4, 2), (0, 3, 4, 1, 2), (2, 0, 4, 2, 3), (2, 3, 0, 0, 4)]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("full,resets,lengths", [(True, True, True), (False, False, False), (True, False, True), (False, True, False)])
@pytest.mark.parametrize("sizes", SCAN_SIZES)
def test_scan(numpy_backend, sizes, full, resets, lengths, dtype):
    check_scan(numpy_backend, sizes, dtype, full, resets, lengths)


def check_scan_leaves_unread(backend, sizes, dtype):
    """What is behind a row's end, and states before a reset, may be anything; nothing of it passes."""
    given, grad, grad_state = scan_inputs(sizes, dtype, 4)
    time = sizes[1]
    ends, middle = np.clip(given["lengths"], 0, time), time // 2
    ends[0] = given["lengths"][0] = time
    given["resets"][:, middle] = True
    spoiled = {k: None if v is None else v.copy() for k, v in given.items()}
    bad_grad, bad_initial = grad.copy(), spoiled["initial"]
    for row, end in enumerate(ends):
        for name in ("x", "delta", "b", "c", "gate"):
            spoiled[name][row, end:] = np.nan if row % 2 else np.inf
        bad_grad[row, end:] = np.nan
    bad_initial[0] = np.inf
    results = []
    for values, d in ((given, grad), (spoiled, bad_grad)):
        arrays, options = put_scan(backend, values)
        results.append([p.asnumpy(v) for v in p.nn.selective_scan(*arrays, **options)])
        arrays[7] = p.asarray(given["initial"], backend=backend)  # gradients of states that are infinite are NaN
        found = p.nn.selective_scan_grad(p.asarray(d, backend=backend), *arrays, **options, grad_state=p.asarray(grad_state, backend=backend))
        results[-1] += [p.asnumpy(v) for v in found]
    one, two = results
    np.testing.assert_array_equal(one[0][:, middle:], two[0][:, middle:])
    np.testing.assert_array_equal(one[1][0], two[1][0])
    for a, b in zip(one[2:], two[2:]):
        np.testing.assert_array_equal(a, b)
    for row, end in enumerate(ends):
        for array in (two[0], two[2], two[3], two[5], two[6], two[8]):
            assert not array[row, end:].any()
        if end == 0:
            np.testing.assert_array_equal(two[10][row], grad_state[row])


@pytest.mark.parametrize("dtype", FLOATS)
def test_scan_leaves_unread(numpy_backend, dtype):
    check_scan_leaves_unread(numpy_backend, (4, 31, 6, 2, 3), dtype)


def check_scan_goes_on(backend, dtype, sizes=(2, 9, 6, 2, 4)):
    """From the last states on, by sequences and by single tokens, as one call does."""
    given, _, _ = scan_inputs(sizes, dtype, 2, lengths=False)
    arrays, options = put_scan(backend, given)
    want = blocks.selective_scan(**given)
    time, state = sizes[1], given["initial"]
    for low, high in ((0, 1), (1, 4), (4, time)):
        part = {k: v[:, low:high] if k in ("x", "delta", "b", "c", "gate", "resets") else v for k, v in given.items()}
        part["initial"] = state
        some, more = put_scan(backend, part)
        y, last = p.nn.selective_scan(*some, **more)
        within(y, want[0][:, low:high], dtype)
        state = p.asnumpy(last)
    within(last, want[1], dtype)
    given["resets"] = None
    want = blocks.selective_scan(**given)
    state = p.asarray(given["initial"], backend=backend)
    at = [p.asarray(given[k], backend=backend) for k in ("x", "delta", "a_log", "b", "c", "skip", "gate", "delta_bias")]
    for t in range(time):
        x, delta, b, c, gate = (at[i][:, t] for i in (0, 1, 3, 4, 6))
        y, state = p.nn.selective_scan_step(x, delta, at[2], b, c, state, at[5], gate, delta_bias=at[7])
        within(y, want[0][:, t], dtype)
    within(state, want[1], dtype)


@pytest.mark.parametrize("dtype", FLOATS)
def test_scan_goes_on(numpy_backend, dtype):
    check_scan_goes_on(numpy_backend, dtype)


def test_scan_gradients_match_differences(numpy_backend):
    given, grad, grad_state = scan_inputs((2, 5, 4, 2, 2), np.float64, 5, lengths=False)
    given["resets"] = np.zeros((2, 5), bool)
    given["resets"][0, 3] = True
    given["lengths"] = np.array([5, 3])
    names = [n for n in SCAN_NAMES if given[n] is not None and n not in ("resets", "lengths")]

    def value(values):
        arrays, options = put_scan(numpy_backend, {**given, **dict(zip(names, values))})
        y, last = p.nn.selective_scan(*arrays, **options)
        return float((grad * p.asnumpy(y)).sum() + (grad_state * p.asnumpy(last)).sum())

    arrays, options = put_scan(numpy_backend, given)
    found = p.nn.selective_scan_grad(p.asarray(grad), *arrays, **options, grad_state=p.asarray(grad_state))
    for which, name in enumerate(names):
        want = differences(value, [given[n] for n in names], which)
        # Central differences: third derivatives of order 100 times step^2, rounding over the step.
        np.testing.assert_allclose(p.asnumpy(getattr(found, name)), want, atol=2e-8, err_msg=name)


def test_scan_refusals(numpy_backend):
    f = p.nn.selective_scan

    def zeros(*shape):
        return p.zeros(shape, dtype="float32")

    x, a, b = zeros(2, 3, 4), zeros(4, 5), zeros(2, 3, 2, 5)
    f(x, x, a, b, b)
    for bad in (zeros(4), zeros(3, 5), zeros(4, 0), zeros(4, 257)):
        with pytest.raises(ValueError, match="a_log"):
            f(x, x, bad, b, b)
    for bad in (zeros(2, 3, 5), zeros(2, 4, 2, 5), zeros(2, 3, 2, 4)):
        with pytest.raises(ValueError, match="b must"):
            f(x, x, a, bad, bad)
    with pytest.raises(ValueError, match="do not divide"):
        f(x, x, a, zeros(2, 3, 3, 5), zeros(2, 3, 3, 5))
    with pytest.raises(ValueError, match="do not divide"):
        f(x, x, a, zeros(2, 3, 0, 5), zeros(2, 3, 0, 5))
    with pytest.raises(ValueError, match="without channels"):
        f(zeros(2, 3, 0), zeros(2, 3, 0), zeros(0, 5), b, b)
    with pytest.raises(ValueError, match="c must"):
        f(x, x, a, b, zeros(2, 3, 1, 5))
    with pytest.raises(ValueError, match="delta must"):
        f(x, zeros(2, 3, 1), a, b, b)
    for name, bad in (("skip", zeros(2, 4)), ("gate", zeros(4)), ("initial", zeros(2, 4)), ("delta_bias", zeros(3)), ("resets", np.zeros(2, bool)), ("lengths", np.zeros((2, 3), int))):
        with pytest.raises(ValueError, match=name):
            f(x, x, a, b, b, **{name: bad})
    with pytest.raises(p.UnsupportedDtypeError):
        f(x, p.zeros((2, 3, 4), dtype="float64"), a, b, b)
    with pytest.raises(ValueError, match="grad must"):
        p.nn.selective_scan_grad(a, x, x, a, b, b)
    with pytest.raises(ValueError, match="grad_state"):
        p.nn.selective_scan_grad(x, x, x, a, b, b, grad_state=x)
    with pytest.raises(ValueError, match="state must"):
        p.nn.selective_scan_step(x[:, 0], x[:, 0], a, b[:, 0], b[:, 0], x)
    with pytest.raises(ValueError):
        p.nn.selective_scan_step(zeros(), zeros(), a, b, b, x)
    with pytest.raises(NotImplementedError, match="not captured"):
        p.compile(lambda x, a, b: f(x, x, a, b, b)[0])(x, a, b)


# ---- residual stream and norms -------------------------------------------------------

GATES = {"none": lambda lead: None, "channel": lambda lead: (), "sequence": lambda lead: lead[:1] + (1,) * (len(lead) - 1), "token": lambda lead: lead}


def norm_inputs(lead, channels, dtype, seed, gate, post):
    rng = np.random.default_rng(seed)

    def normal(*shape):
        return rng.standard_normal(shape).astype(dtype)

    axes = GATES[gate](lead)
    x, residual, ds, dn = (normal(*lead, channels) for _ in range(4))
    return x, 3 * residual, normal(channels), normal(channels) if post else None, None if axes is None else normal(*axes, channels), ds, dn


def check_norm(backend, lead, channels, dtype, gate, post, scale=0.7, eps=1e-6):
    x, residual, weight, post_weight, gates, ds, dn = norm_inputs(lead, channels, dtype, channels + len(lead), gate, post)
    xs, res, ws, pw, gs, dss, dns = put(backend, x, residual, weight, post_weight, gates, ds, dn)
    options = dict(post_weight=pw, gate=gs, scale=scale, eps=eps)
    rows = int(np.prod(lead))
    divide = 1 if gates is None or gate == "token" else rows // (lead[0] if gate == "sequence" and lead else 1) if rows else 1
    flat = lambda v: v.reshape(rows, channels)  # noqa: E731
    stream, normed = p.nn.residual_norm(xs, res, ws, **options)
    plain = (post_weight, gates, divide, scale, eps)
    for got, want in zip((stream, normed), blocks.residual_norm(flat(x), flat(residual), weight, *plain)):
        assert got.shape == x.shape
        within(got.reshape(rows, channels), want, dtype)
    found = p.nn.residual_norm_grad(dss, dns, xs, stream, ws, **options)
    want = blocks.residual_norm_grad(flat(ds), flat(dn), flat(x), flat(p.asnumpy(stream)), weight, *plain)
    for like, got, value in zip((x, x, weight, post_weight, gates), found, want):
        assert (got is None) == (like is None)
        if got is not None:
            assert got.shape == like.shape
            within(got.reshape(value.value.shape), value, dtype)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate", list(GATES))
@pytest.mark.parametrize("lead,channels", [((), 1), ((3,), 7), ((2, 5), 16), ((2, 3, 2), 33), ((4,), 1)])
def test_norm(numpy_backend, lead, channels, gate, post, dtype):
    check_norm(numpy_backend, lead, channels, dtype, gate, post)


@pytest.mark.parametrize("gate", list(GATES))
@pytest.mark.parametrize("lead", [(0,), (0, 3), (3, 0)])
def test_norm_of_no_rows(numpy_backend, lead, gate):
    check_norm_of_no_rows(numpy_backend, lead, gate)


def check_norm_of_no_rows(backend, lead, gate):
    x, residual, weight, post_weight, gates, ds, dn = put(backend, *norm_inputs(lead, 4, np.float32, 0, gate, True))
    for got in p.nn.residual_norm(x, residual, weight, post_weight=post_weight, gate=gates):
        assert got.shape == lead + (4,)
    found = p.nn.residual_norm_grad(ds, dn, x, residual, weight, post_weight=post_weight, gate=gates)
    for like, got in zip((x, x, weight, post_weight, gates), found):
        if like is not None:
            assert got.shape == like.shape and not p.asnumpy(got).any()


def test_norm_gradients_match_differences(numpy_backend):
    for gate in GATES:
        x, residual, weight, post_weight, gates, ds, dn = norm_inputs((2, 3), 5, np.float64, 1, gate, True)

        def value(given):
            x, residual, weight, post_weight, gates = put(numpy_backend, *given)
            found = p.nn.residual_norm(x, residual, weight, post_weight=post_weight, gate=gates, scale=0.3, eps=0.1)
            return sum(float((d * p.asnumpy(v)).sum()) for d, v in zip((ds, dn), found))

        given = [x, residual, weight, post_weight, gates]
        arrays = put(numpy_backend, *given)
        options = dict(post_weight=arrays[3], gate=arrays[4], scale=0.3, eps=0.1)
        stream = p.nn.residual_norm(*arrays[:3], **options)[0]
        found = p.nn.residual_norm_grad(p.asarray(ds), p.asarray(dn), arrays[0], stream, arrays[2], **options)
        for which, got in enumerate(found):
            if got is not None:
                # Central differences: third derivatives of order 10 times step^2, rounding over the step.
                np.testing.assert_allclose(p.asnumpy(got), differences(value, given, which), atol=1e-8)


def test_norm_refusals(numpy_backend):
    f = p.nn.residual_norm

    def zeros(*shape):
        return p.zeros(shape, dtype="float32")

    x, w = zeros(2, 3, 4), zeros(4)
    for bad in (zeros(), zeros(3, 0)):
        with pytest.raises(ValueError, match="none of it empty"):
            f(bad, bad, w)
    with pytest.raises(ValueError, match="weight"):
        f(x, x, zeros(3))
    with pytest.raises(ValueError, match="residual"):
        f(x, zeros(3, 4), w)
    with pytest.raises(ValueError, match="post_weight"):
        f(x, x, w, post_weight=zeros(1))
    for bad in (zeros(2, 3, 1), zeros(1, 3, 4), zeros(3, 4), zeros(), zeros(1, 2, 3, 4)):
        with pytest.raises(ValueError, match="gate"):
            f(x, x, w, gate=bad)
    f(x, x, w, gate=zeros(1, 1, 4))
    for eps in (0.0, -1.0, 1e-40, np.nan, np.inf):
        with pytest.raises(ValueError):
            f(x, x, w, eps=eps)
    for scale in (np.nan, np.inf):
        with pytest.raises(ValueError, match="scale"):
            f(x, x, w, scale=scale)
    with pytest.raises(p.UnsupportedDtypeError):
        f(x, x, p.zeros((4,), dtype="float64"))
    for at in range(2):
        grads = [x, x]
        grads[at] = w
        with pytest.raises(ValueError, match="grad_"):
            p.nn.residual_norm_grad(*grads, x, x, w)
    with pytest.raises(ValueError, match="stream"):
        p.nn.residual_norm_grad(x, x, x, w, w)
    with pytest.raises(NotImplementedError, match="not captured"):
        p.compile(lambda x, w: f(x, x, w)[0])(x, w)
