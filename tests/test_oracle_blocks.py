"""The oracle of the convolution, the scan, the residual norms and the distillation loss (oracle/blocks.py): closed
forms, central differences of its own values, and mistakes that its bounds have to find."""

import numpy as np
import pytest

import openpacho as p
from oracle import blocks
from test_nn_blocks import SCAN_NAMES, conv_inputs, norm_inputs, put_scan, scan_inputs, within
from test_nn_distillation import inputs as distillation_inputs
from test_nn_losses import within as within_units

WIDE = blocks.WIDE
CLOSE = dict(rtol=1e-17, atol=1e-17)  # some roundings of 64 bits of fraction, 5.4e-20 each


# ---- closed forms --------------------------------------------------------------------


def test_conv_closed_forms():
    # An impulse leaves the taps from the last to the first; a reset hides it, a row's end cuts them off.
    weight = np.array([[2.0, 3.0, 5.0]])
    x = np.zeros((3, 5, 1))
    x[:, 1] = 1
    resets = np.zeros((3, 5), bool)
    resets[1, 2] = True
    y, last = blocks.causal_conv(x, weight, np.array([7.0]), resets=resets, lengths=[5, 5, 3])
    np.testing.assert_array_equal(y.value[..., 0], [[7, 12, 10, 9, 7], [7, 12, 7, 7, 7], [7, 12, 10, 0, 0]])
    np.testing.assert_array_equal(last[..., 0], [[0, 0], [0, 0], [1, 0]])
    # Carried inputs; silu of 0 and of log 3, whose sigmoid is 3/4.
    y, last = blocks.causal_conv(np.zeros((1, 2, 1)), weight, initial=np.array([[[0.0], [np.log(3.0) / 3]]]), activation="silu")
    np.testing.assert_allclose(y.value[0, :, 0], [np.log(WIDE(3)) * 0.75, np.log(WIDE(3)) * 2 / 3 / (1 + WIDE(3) ** (-WIDE(2) / 3))], rtol=1e-15)
    assert not last.any()


def test_conv_gradients_closed_forms():
    # Every gradient is 1: dx counts the taps that see an input, dw sums what each tap saw, dbias counts steps.
    x = np.arange(1.0, 5.0).reshape(1, 4, 1)
    dx, dw, db, di = blocks.causal_conv(x, np.array([[2.0, 3.0, 5.0]]), initial=np.array([[[10.0], [20.0]]]), grad=np.ones((1, 4, 1)))
    np.testing.assert_array_equal(dx.value[0, :, 0], [10, 10, 8, 5])
    np.testing.assert_array_equal(dw.value, [[10 + 20 + 1 + 2, 20 + 1 + 2 + 3, 1 + 2 + 3 + 4]])
    np.testing.assert_array_equal(db.value, [4])
    np.testing.assert_array_equal(di.value[0, :, 0], [2, 5])


def halving(time, **more):
    """delta = 0 gives dt = log 2, a_log = 0 a decay of 1/2."""
    one, zero = np.ones((1, time, 1)), np.zeros((1, time, 1))
    return dict(x=one, delta=zero, a_log=np.zeros((1, 1)), b=np.ones((1, time, 1, 1)), c=np.ones((1, time, 1, 1)), **more)


def test_scan_closed_forms():
    log2, steps = np.log(WIDE(2)), np.arange(1, 7)
    # h_t = 2 log 2 (1 - 2^-t), and 2^-t of a carried state.
    y, last = blocks.selective_scan(**halving(6, initial=np.full((1, 1, 1), 3.0)))
    want = 2 * log2 * (1 - WIDE(2.0) ** -steps) + 3 * WIDE(2.0) ** -steps
    np.testing.assert_allclose(y.value[0, :, 0], want, **CLOSE)
    np.testing.assert_allclose(last.value[0, 0, 0], want[-1], **CLOSE)
    # From a reset on as from the start; nothing behind the end; skip; silu(log 3) = 3/4 log 3.
    resets = np.zeros((1, 6), bool)
    resets[0, 2] = True
    gate = np.full((1, 6, 1), np.log(3.0))
    y, last = blocks.selective_scan(**halving(6, initial=np.full((1, 1, 1), 3.0), resets=resets, lengths=[5], skip=np.array([0.5]), gate=gate))
    again = 2 * log2 * (1 - WIDE(2.0) ** -steps)
    want = np.array([*want[:2], *again[:3], -0.5]) + 0.5
    np.testing.assert_allclose(y.value[0, :, 0], want * 0.75 * np.log(WIDE(3)), rtol=1e-15, atol=1e-17)
    np.testing.assert_allclose(last.value[0, 0, 0], again[2], **CLOSE)


def test_scan_gradients_closed_forms():
    # Of the last state alone: e_t = 2^-(6 - t). da = -r sum e_t h_{t-1} dt, with h_t = 3 2^-t where x is 0.
    given = halving(6, initial=np.full((1, 1, 1), 3.0))
    given["x"] = np.zeros((1, 6, 1))
    found = blocks.selective_scan(**given, grad=np.zeros((1, 6, 1)), grad_state=np.ones((1, 1, 1)))
    dx, d_delta, da, db, dc, d_skip, d_gate, d_bias, d_initial = found
    log2, after = np.log(WIDE(2)), WIDE(2.0) ** -np.arange(5, -1, -1)
    np.testing.assert_allclose(d_initial.value[0, 0, 0], WIDE(2.0) ** -6, **CLOSE)
    np.testing.assert_allclose(dx.value[0, :, 0], after * log2, **CLOSE)
    np.testing.assert_allclose(da.value[0, 0], -log2 * 6 * 3 * WIDE(2.0) ** -6, **CLOSE)
    # ddt_t = -e_t h_{t-1}/2, the slope of softplus at 0 is 1/2.
    np.testing.assert_allclose(d_delta.value[0, :, 0], np.full(6, -3 * WIDE(2.0) ** -6 / 2), **CLOSE)
    np.testing.assert_allclose(d_bias.value, [-18 * WIDE(2.0) ** -6 / 2], **CLOSE)
    assert not db.value.any() and not dc.value.any() and not d_skip.value.any() and d_gate is None


def test_norm_closed_forms():
    # A single channel: rms(v) = v / sqrt(v^2 + eps), whose slope is eps / (v^2 + eps)^(3/2).
    x, residual, eps = np.array([[3.0], [-2.0]]), np.array([[1.0], [4.0]]), 7.0
    unit = x / np.sqrt(x.astype(WIDE) ** 2 + eps)
    stream, normed = blocks.residual_norm(x, residual, np.array([2.0]), np.array([5.0]), np.array([0.5]), 2, 4.0, eps)
    want = residual + 4 * 0.5 * unit * 5
    np.testing.assert_allclose(stream.value, want, **CLOSE)
    np.testing.assert_allclose(normed.value, 2 * want / np.sqrt(want**2 + eps), **CLOSE)
    given = np.array([[2.0], [-1.0]])
    slope, inner = eps / (given.astype(WIDE) ** 2 + eps) ** 1.5, eps / (x.astype(WIDE) ** 2 + eps) ** 1.5
    ds, dn = np.array([[1.0], [0.5]]), np.array([[3.0], [-1.0]])
    dx, d, d_weight, d_post, d_gate = blocks.residual_norm_grad(ds, dn, x, given, np.array([2.0]), np.array([5.0]), np.array([0.5]), 2, 4.0, eps)
    want = ds + dn * 2 * slope
    np.testing.assert_allclose(d.value, want, **CLOSE)
    np.testing.assert_allclose(dx.value, want * 4 * 0.5 * 5 * inner, **CLOSE)
    np.testing.assert_allclose(d_weight.value, [(dn * given / np.sqrt(given.astype(WIDE) ** 2 + eps)).sum()], **CLOSE)
    np.testing.assert_allclose(d_post.value, [(want * 2 * unit).sum()], **CLOSE)
    np.testing.assert_allclose(d_gate.value, [[(want * 4 * unit * 5).sum()]], **CLOSE)


def test_distillation_closed_forms():
    # q = (1, 1, 2) / 4; the list (1/3, 2/3) of the first and the last; with the rest (1/4, 1/2) and 1/4 of the second.
    z, t = np.log(np.array([[1.0, 1.0, 2.0]])), np.log(np.array([[1.0, 2.0]]))
    (loss, losses, grad), _ = blocks.distillation_loss(z, np.array([[0, 2]]), t)
    np.testing.assert_allclose(losses, [np.log(4 / 3)], rtol=1e-15)
    np.testing.assert_allclose(grad, [[0.25 - 1 / 3, 0.25, 0.5 - 2 / 3]], rtol=1e-14)
    (loss, losses, grad), _ = blocks.distillation_loss(z, np.array([[0, 2]]), t, np.zeros(1), count=5)
    np.testing.assert_allclose([loss, *losses, *grad[0]], np.zeros(5), atol=1e-16)
    # A temperature of 2 takes the square roots of both sides; the gradient is half as large.
    (loss, losses, grad), _ = blocks.distillation_loss(2 * z, np.array([[0, 2]]), 2 * t, temperature=2.0)
    np.testing.assert_allclose(losses, [np.log(4 / 3)], rtol=1e-15)
    np.testing.assert_allclose(grad, np.array([[0.25 - 1 / 3, 0.25, 0.5 - 2 / 3]]) / 2, rtol=1e-14)


# ---- differences -----------------------------------------------------------------------

STEP = WIDE(1e-6)


def differences(value, given):
    """Central differences of value() by the elements of `given`, in extended precision: what third derivatives of
    order 100 leave is 1e-10, what rounding does 1e-13."""
    found = np.empty(given.shape, WIDE)
    for at in np.ndindex(given.shape):
        ends = []
        for sign in (1, -1):
            moved = given.astype(WIDE)
            moved[at] += sign * STEP
            ends.append(value(moved))
        found[at] = (ends[0] - ends[1]) / (2 * STEP)
    return found


def agree(found, want, name):
    np.testing.assert_allclose(found.astype(np.float64), want.astype(np.float64), rtol=0, atol=1e-9, err_msg=name)


@pytest.mark.parametrize("activation", [None, "silu"])
def test_conv_gradients_match_differences(activation):
    x, weight, bias, initial, starts, _, d = conv_inputs((2, 5, 2, 3), np.float64, 3, spoiled=False)
    given, ends = {"x": x, "weight": weight, "bias": bias, "initial": initial}, np.array([5, 3])
    found = blocks.causal_conv(**given, resets=starts, lengths=ends, activation=activation, grad=d)
    for name, got in zip(given, found):
        def value(moved):
            return (d * blocks.causal_conv(**{**given, name: moved}, resets=starts, lengths=ends, activation=activation)[0].value).sum()

        agree(got.value, differences(value, given[name]), name)


def test_scan_gradients_match_differences():
    given, grad, grad_state = scan_inputs((2, 4, 4, 2, 2), np.float64, 3)
    given["resets"][:], given["lengths"] = False, np.array([4, 2])
    given["resets"][0, 2] = True
    names = ("x", "delta", "a_log", "b", "c", "skip", "gate", "delta_bias", "initial")
    found = blocks.selective_scan(**given, grad=grad, grad_state=grad_state)
    for name, got in zip(names, found):
        def value(moved):
            y, last = blocks.selective_scan(**{**given, name: moved})
            return (grad * y.value).sum() + (grad_state * last.value).sum()

        agree(got.value, differences(value, given[name]), name)


def test_norm_gradients_match_differences():
    x, residual, weight, post, gate, ds, dn = norm_inputs((4,), 3, np.float64, 1, "channel", True)
    given, options = {"x": x, "residual": residual, "weight": weight, "post_weight": post, "gate": gate}, dict(divide=4, scale=0.3, eps=0.1)
    stream = blocks.residual_norm(**given, **options)[0].value
    found = blocks.residual_norm_grad(ds, dn, x, stream, weight, post, gate, **options)
    for name, got in zip(given, found):
        def value(moved):
            a, b = blocks.residual_norm(**{**given, name: moved}, **options)
            return (ds * a.value).sum() + (dn * b.value).sum()

        agree(got.value.reshape(given[name].shape), differences(value, given[name]), name)


@pytest.mark.parametrize("rest", [True, False])
def test_distillation_gradients_match_differences(rest):
    z, order, listed, others, _ = distillation_inputs(4, 6, 3, np.float64, 2, rest, False)
    mask = np.array([True, True, False, True])
    (_, _, grad), _ = blocks.distillation_loss(z, order, listed, others, mask, 1.5)
    agree(grad, differences(lambda moved: blocks.distillation_loss(moved, order, listed, others, mask, 1.5)[0][0], z), "logits")


# ---- planted mistakes --------------------------------------------------------------------


def refused(check, *args):
    with pytest.raises(AssertionError):
        check(*args)


def one_off(values, by):
    """The values as they are, but for one of middle size of those that are not 0."""
    values = np.array(values)
    flat = values.reshape(-1)
    there = np.flatnonzero(flat)
    flat[there[np.argsort(np.abs(flat[there]))[len(there) // 2]]] *= 1 + by
    return p.asarray(values)


# One value that is off by 2^12 units of rounding (2^-24, 2^-53), 2.4e-4 and 4.5e-13 of it; where the values are sums whose
# terms cancel, by 2^14.
MISTAKE = {np.float32: 2.0**-12, np.float64: 2.0**-41}


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_conv_mistakes_are_found(dtype):
    x, weight, bias, initial, starts, ends, d = conv_inputs((2, 12, 5, 4), dtype, 5, spoiled=False)
    starts[:], ends[:] = False, (12, 9)
    starts[:, 5] = True
    options = dict(initial=initial, resets=starts, lengths=ends, activation="silu")
    want, last = blocks.causal_conv(x, weight, bias, **options)
    right = p.nn.causal_conv(x, p.asarray(weight), bias, **options)
    within(right[0], want, dtype)
    refused(within, one_off(p.asnumpy(right[0]), MISTAKE[dtype]), want, dtype)
    for wrong in (
        dict(weight=weight[:, ::-1].copy()), dict(bias=None), dict(initial=None), dict(resets=np.roll(starts, 1, 1)), dict(resets=None),
        dict(lengths=ends - 1), dict(activation=None),
    ):  # fmt: skip
        given = {**dict(weight=weight, bias=bias), **options, **wrong}
        y, end = p.nn.causal_conv(p.asarray(x), given.pop("weight"), given.pop("bias"), **given)
        refused(within, y, want, dtype)
    grads = blocks.causal_conv(x, weight, bias, **options, grad=d)
    found = p.nn.causal_conv_grad(d, p.asarray(x), weight, bias, **options)
    other = p.nn.causal_conv_grad(d, p.asarray(x), weight, bias, **{**options, "activation": None})
    for got, wrong, value in zip(found, other, grads):
        within(got, value, dtype)
        refused(within, wrong, value, dtype)
        refused(within, one_off(p.asnumpy(got), MISTAKE[dtype]), value, dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_scan_mistakes_are_found(dtype):
    given, grad, grad_state = scan_inputs((2, 12, 4, 2, 3), dtype, 8)
    given["resets"][:], given["lengths"] = False, np.array([12, 9])
    given["resets"][:, 5] = True
    want = blocks.selective_scan(**given)
    grads = blocks.selective_scan(**given, grad=grad, grad_state=grad_state)

    def run(values, gradient=False):
        arrays, options = put_scan(None, values)
        if gradient:
            return p.nn.selective_scan_grad(p.asarray(grad), *arrays, **options, grad_state=grad_state)
        return p.nn.selective_scan(*arrays, **options)

    right = run(given)
    for got, value in zip(right, want):
        within(got, value, dtype)
    refused(within, one_off(p.asnumpy(right[0]), MISTAKE[dtype]), want[0], dtype)
    turned = {**given, "b": given["c"], "c": given["b"]}
    groups = {**given, "b": given["b"][:, :, ::-1].copy(), "c": given["c"][:, :, ::-1].copy()}
    for wrong in (
        turned, groups, {**given, "skip": None}, {**given, "gate": None}, {**given, "initial": None}, {**given, "delta_bias": None},
        {**given, "resets": np.roll(given["resets"], 1, 1)}, {**given, "lengths": given["lengths"] - 1}, {**given, "a_log": given["a_log"] + dtype(0.01)},
    ):  # fmt: skip
        refused(within, run(wrong)[0], want[0], dtype)
    found = run(given, True)
    for name, got, value in zip(found._fields, found, grads):
        within(got, value, dtype)
        refused(within, one_off(p.asnumpy(got), 4 * MISTAKE[dtype]), value, dtype)
    for got, value in zip(run(turned, True)[:5], grads):
        refused(within, got, value, dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_norm_mistakes_are_found(dtype):
    x, residual, weight, post, gate, ds, dn = norm_inputs((6,), 40, dtype, 3, "channel", True)
    options = dict(post_weight=post, gate=gate, scale=0.7, eps=1e-2)
    want = blocks.residual_norm(x, residual, weight, post, gate, 6, 0.7, 1e-2)
    right = p.nn.residual_norm(p.asarray(x), residual, weight, **options)
    for got, value in zip(right, want):
        within(got, value, dtype)
        refused(within, one_off(p.asnumpy(got), MISTAKE[dtype]), value, dtype)
    for wrong in (dict(post_weight=None), dict(gate=None), dict(scale=0.71), dict(eps=1.1e-2)):
        refused(within, p.nn.residual_norm(p.asarray(x), residual, weight, **{**options, **wrong})[1], want[1], dtype)
    stream = p.asnumpy(right[0])
    grads = blocks.residual_norm_grad(ds, dn, x, stream, weight, post, gate, 6, 0.7, 1e-2)
    found = p.nn.residual_norm_grad(ds, dn, p.asarray(x), stream, weight, **options)
    swapped = p.nn.residual_norm_grad(dn, ds, p.asarray(x), stream, weight, **options)
    for got, wrong, value in zip(found, swapped, grads):
        shape = value.value.shape
        within(got.reshape(shape), value, dtype)
        refused(within, wrong.reshape(shape), value, dtype)
        refused(within, one_off(p.asnumpy(got).reshape(shape), MISTAKE[dtype]), value, dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_distillation_mistakes_are_found(dtype):
    z, order, listed, others, mask = distillation_inputs(9, 30, 6, dtype, 4)
    values, units = blocks.distillation_loss(z, order, listed, others, mask, 1.5)
    right = p.nn.distillation_loss_grad(p.asarray(z), order, listed, others, mask=mask, temperature=1.5)
    for got, want, unit in zip(right, values, units):
        within_units(got, want, unit, dtype)
    for got, want, unit in zip(right[1:], values[1:], units[1:]):
        refused(within_units, one_off(p.asnumpy(got), 4 * MISTAKE[dtype]), want, unit, dtype)
    for wrong in (dict(teacher_rest=None), dict(temperature=1.51), dict(count=len(mask)), dict(teacher_logits=np.roll(listed, 1, 1))):
        given = {**dict(teacher_logits=listed, teacher_rest=others, mask=mask, temperature=1.5), **wrong}
        found = p.nn.distillation_loss_grad(p.asarray(z), order, **given)
        refused(within_units, found[2], values[2], units[2], dtype)
