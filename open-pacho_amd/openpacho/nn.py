"""Operators of model training and serving: recurrences, convolutions and scans over time, residual norms,
losses from logits, AdamW.

Each works on resident arrays of one backend, float32 or float64 throughout,
and returns new arrays; gradients are functions of their own, since arrays
carry no history. Host values given in an array's place are converted to the
dtype of the call's arrays and uploaded. ``compile`` and ``fuse`` do not capture
these operators: call them between compiled functions.

    h = nn.gated_recurrence(x, gate, initial, resets=starts)
    loss, log_probs, d_logits = nn.policy_loss_grad(logits, actions, old, advantages, mask=mask)
    dx, d_gate, d_initial = nn.gated_recurrence_grad(d_h, x, gate, h, initial, resets=starts)
    params, state = nn.adamw(params, grads, state, learning_rate=3e-4)

    u, inputs = nn.causal_conv(x, weight, bias, activation="silu", resets=starts, lengths=lengths)
    y, states = nn.selective_scan(u, delta, a_log, b, c, skip, gate, delta_bias=bias, resets=starts, lengths=lengths)
    stream, normed = nn.residual_norm(y @ w_out, stream, weight)
    loss, losses, d_logits = nn.distillation_loss_grad(logits, indices, teacher_logits, teacher_rest, mask=mask)
    d = nn.selective_scan_grad(d_y, u, delta, a_log, b, c, skip, gate, delta_bias=bias, resets=starts, lengths=lengths)
    y, states = nn.selective_scan_step(u, delta, a_log, b, c, states, skip, gate, delta_bias=bias)  # one token
"""

import math
import operator
from math import prod
from typing import NamedTuple

import numpy as np

from . import _array as xp
from .backends import _DEFAULT
from .exceptions import BackendMismatchError, UnsupportedDtypeError

_FLOATS = (np.dtype("float32"), np.dtype("float64"))
_TINY = {dtype: float(np.finfo(dtype).tiny) for dtype in _FLOATS}
_INDICES = (np.dtype("int32"), np.dtype("int64"))
_BOOL = np.dtype("bool")


# ---- arguments -----------------------------------------------------------------


def _refuse_capture(what, backend):
    if backend._is_tracing or _DEFAULT.get()._is_tracing:
        raise NotImplementedError(f"{what} is not captured; call it between compiled functions")


class _Operands:
    """The arrays of one call: their backend, and their float dtype, which the first one gives that is no host value."""

    __slots__ = ("what", "backend", "dtype")

    def __init__(self, what, lead, *others):
        self.what, self.backend = what, xp._common_backend((lead, *others)) if not isinstance(lead, xp.ndarray) else lead._backend
        for value in others:
            if value is not None and isinstance(value, xp.ndarray) and value._backend is not self.backend:
                raise BackendMismatchError("Arrays belong to different backends/devices; use to_backend()")
        _refuse_capture(what, self.backend)
        if isinstance(lead, xp.ndarray):
            self.dtype = lead._dtype
        else:
            given = [v._dtype for v in others if isinstance(v, xp.ndarray) and v._dtype in _FLOATS]
            self.dtype = given[0] if given else np.asarray(lead).dtype
        if self.dtype not in _FLOATS:
            raise UnsupportedDtypeError(f"{what} requires float32 or float64, got {self.dtype}")

    def array(self, name, value, shape=None, dtypes=None):
        """`value` as an array of the call's dtype (or one of `dtypes`) and of `shape`."""
        dtypes = (self.dtype,) if dtypes is None else dtypes
        if not isinstance(value, xp.ndarray):
            host = np.asarray(value)
            value = xp.asarray(host if host.dtype in dtypes else self._converted(name, host, dtypes[-1]), backend=self.backend)
        if value._dtype not in dtypes:
            wanted = " or ".join(map(str, dtypes))
            raise UnsupportedDtypeError(f"{self.what}: {name} must be {wanted}, got {value.dtype}")
        if shape is not None and value._shape != shape:
            raise ValueError(f"{self.what}: {name} must have shape {shape}, got {value.shape}")
        return value

    def _converted(self, name, host, dtype):
        if host.dtype.kind not in ("b" if dtype == _BOOL else "iu" if dtype.kind == "i" else "fiu"):
            raise UnsupportedDtypeError(f"{self.what}: {name} must be {dtype}, got {host.dtype}")
        return host.astype(dtype)

    def optional(self, name, value, shape, dtypes=None):
        return None if value is None else self.array(name, value, shape, dtypes)

    def broadcast(self, name, value, shape):
        """`value`, which has to broadcast to `shape`."""
        value = self.array(name, value)
        if value._shape != shape and not (shape and value._shape == shape[:-1] + (1,)):
            try:
                whole = np.broadcast_shapes(value._shape, shape) == shape
            except ValueError:
                whole = False
            if not whole:
                raise ValueError(f"{self.what}: {name} of shape {value.shape} does not broadcast to {shape}")
        return value

    def result(self, data, shape):
        return _wrapped(data, shape, self.dtype, self.backend)


def _wrapped(data, shape, dtype, backend):
    """ndarray._wrap of storage whose shape and dtype are as an array keeps them."""
    array = object.__new__(xp.ndarray)
    array._data, array._shape, array._dtype, array._backend = data, shape, dtype, backend
    return array


def _number(what, value, least=None, below=None, infinite=False):
    if type(value) is float and least == 0 and 0 <= value < (math.inf if below is None else below):
        return value
    value = float(value)
    if math.isnan(value) or (math.isinf(value) and not infinite):
        raise ValueError(f"{what} must be a finite number")
    if (least is not None and value < least) or (below is not None and value >= below):
        raise ValueError(f"{what} is out of range: {value}")
    return value


def _positive(what, value):
    value = _number(what, value)
    if value <= 0:
        raise ValueError(f"{what} must be positive")
    return value


# ---- gated recurrence ----------------------------------------------------------


def _gates_divide(what, channels, gates):
    if channels and (not gates or channels % gates):
        raise ValueError(f"{what}: {gates} gates do not divide {channels} channels")
    if not channels and gates:
        raise ValueError(f"{what}: {gates} gates without channels")


def _recurrence_operands(what, x, gate, initial, resets, *others):
    ops = _Operands(what, x, gate, initial, resets, *others)
    x = ops.array("x", x)
    if len(x._shape) < 2:
        raise ValueError(f"{what}: x must have axes (..., time, channels), got {x.shape}")
    lead, (time, channels) = x._shape[:-2], x._shape[-2:]
    gate = ops.array("gate", gate)
    if not gate._shape or gate._shape[:-1] != x._shape[:-1]:
        raise ValueError(f"{what}: gate must have shape {x.shape[:-1]} and an axis of gates, got {gate.shape}")
    gates = gate._shape[-1]
    if gates != channels:
        _gates_divide(what, channels, gates)
    initial = ops.optional("initial", initial, lead + (channels,))
    resets = ops.optional("resets", resets, lead + (time,), (_BOOL,))
    return ops, x, gate, initial, resets, (prod(lead), time, channels, gates)


def gated_recurrence(x, gate, initial=None, *, resets=None):
    """States ``h_t = a_t h_{t-1} + (1 - a_t) x_t`` with ``a_t = sigmoid(gate_t)``.

    ``x`` has axes (..., time, channels). ``gate`` has a gate per channel, or
    fewer: its last axis divides the channels into heads that share one.
    ``initial`` (..., channels) is the state before the first step, zero if not
    given. Where ``resets`` (..., time) is true the state before that step
    counts as zero, whatever it holds; an infinite state stays so until then, and is
    NaN past a gate whose sigmoid is 0. Returns every state, of x's shape. Equal calls
    give equal bits; a row's rounding may differ beside more or fewer rows.
    """
    ops, x, gate, initial, resets, sizes = _recurrence_operands("gated_recurrence", x, gate, initial, resets)
    return ops.result(ops.backend.gated_recurrence(x, gate, initial, resets, *sizes), x._shape)


def gated_recurrence_step(x, gate, state):
    """The next state of one token: ``gated_recurrence`` of a single step, without its time axis."""
    what = "gated_recurrence_step"
    ops = _Operands(what, x, gate, state)
    x, gate = ops.array("x", x), ops.array("gate", gate)
    if not x._shape or not gate._shape or gate._shape[:-1] != x._shape[:-1]:
        raise ValueError(f"{what}: x and gate must have axes (..., channels) and (..., gates), got {x.shape} and {gate.shape}")
    lead, channels, gates = x._shape[:-1], x._shape[-1], gate._shape[-1]
    _gates_divide(what, channels, gates)
    state = ops.array("state", state, x._shape)
    return ops.result(ops.backend.gated_recurrence(x, gate, state, None, prod(lead), 1, channels, gates), x._shape)


def gated_recurrence_grad(grad, x, gate, h, initial=None, *, resets=None):
    """Gradients (x, gate, initial) of ``gated_recurrence`` whose states ``h`` have the gradient ``grad``.

    A gate that a head shares gets the sum over the head's channels. The third
    gradient is None where no ``initial`` is given.
    """
    what = "gated_recurrence_grad"
    ops, x, gate, initial, resets, sizes = _recurrence_operands(what, x, gate, initial, resets, grad, h)
    grad, h = ops.array("grad", grad, x._shape), ops.array("h", h, x._shape)
    dx, d_gate, d_initial = ops.backend.gated_recurrence_grad(grad, x, gate, h, initial, resets, *sizes)
    first = None if initial is None else ops.result(d_initial, initial._shape)
    return ops.result(dx, x._shape), ops.result(d_gate, gate._shape), first


# ---- causal convolution ----------------------------------------------------------

_MOST_TAPS = 8
_ACTIVATIONS = {None: 0, "silu": 1}


def _conv_weights(ops, channels, weight, bias, activation):
    what = ops.what
    weight = ops.array("weight", weight)
    if len(weight._shape) != 2 or weight._shape[0] != channels:
        raise ValueError(f"{what}: weight must have shape ({channels}, taps), got {weight.shape}")
    taps = weight._shape[1]
    if not 1 <= taps <= _MOST_TAPS:
        raise ValueError(f"{what}: weight must have 1 to {_MOST_TAPS} taps, got {taps}")
    if activation is not None and activation not in _ACTIVATIONS:
        raise ValueError(f"{what}: activation must be None or 'silu', got {activation!r}")
    return weight, ops.optional("bias", bias, (channels,)), taps, _ACTIVATIONS[activation]


def _sequence_operands(what, x, resets, lengths, *others):
    ops = _Operands(what, x, resets, lengths, *others)
    x = ops.array("x", x)
    if len(x._shape) < 2:
        raise ValueError(f"{what}: x must have axes (..., time, channels), got {x.shape}")
    lead, (time, channels) = x._shape[:-2], x._shape[-2:]
    resets = ops.optional("resets", resets, lead + (time,), (_BOOL,))
    lengths = ops.optional("lengths", lengths, lead, _INDICES)
    return ops, x, resets, lengths, lead, (prod(lead), time, channels)


def _conv_operands(what, x, weight, bias, initial, resets, lengths, activation, *others):
    ops, x, resets, lengths, lead, sizes = _sequence_operands(what, x, resets, lengths, weight, bias, initial, *others)
    weight, bias, taps, activation = _conv_weights(ops, sizes[2], weight, bias, activation)
    window = lead + (taps - 1, sizes[2])
    initial = ops.optional("initial", initial, window)
    return ops, x, weight, bias, initial, resets, lengths, window, sizes + (taps, activation)


def causal_conv(x, weight, bias=None, initial=None, *, resets=None, lengths=None, activation=None):
    """A short convolution of each channel over time: (y, last inputs).

    ``y_t = f(bias + sum_k weight[:, k] x_{t - taps + 1 + k})`` of x (..., time,
    channels) with ``weight`` (channels, taps), of 1 to 8 taps; ``f`` is the
    identity or, with ``activation="silu"``, v sigmoid(v). ``initial`` (...,
    taps - 1, channels) are the inputs before the first step, zero if not given.
    Where ``resets`` (..., time) is true, that step and later ones see the inputs
    before it as zero. Rows end after ``lengths`` (...) steps (all of them if not
    given, and at most): what is behind is not read and y is zero there. The
    last inputs (..., taps - 1, channels), as a later step would see them, are
    the ``initial`` of a call that goes on.
    """
    what = "causal_conv"
    ops, x, weight, bias, initial, resets, lengths, window, sizes = _conv_operands(
        what, x, weight, bias, initial, resets, lengths, activation
    )
    y, last = ops.backend.causal_conv(x, weight, bias, initial, resets, lengths, *sizes)
    return ops.result(y, x._shape), ops.result(last, window)


def causal_conv_step(x, weight, state, bias=None, *, activation=None):
    """One token: (y, last inputs) of x (..., channels) after the inputs ``state`` (..., taps - 1, channels)."""
    what = "causal_conv_step"
    ops = _Operands(what, x, weight, state, bias)
    x = ops.array("x", x)
    if not x._shape:
        raise ValueError(f"{what}: x must have axes (..., channels), got {x.shape}")
    lead, channels = x._shape[:-1], x._shape[-1]
    weight, bias, taps, activation = _conv_weights(ops, channels, weight, bias, activation)
    state = ops.array("state", state, lead + (taps - 1, channels))
    y, last = ops.backend.causal_conv(x, weight, bias, state, None, None, prod(lead), 1, channels, taps, activation)
    return ops.result(y, x._shape), ops.result(last, state._shape)


def causal_conv_grad(grad, x, weight, bias=None, initial=None, *, resets=None, lengths=None, activation=None):
    """Gradients (x, weight, bias, initial) of ``causal_conv`` whose y has the gradient ``grad``.

    Those of ``bias`` and ``initial`` are None where they are not given. The
    last inputs' own gradient is not part of it. Equal calls give equal bits.
    """
    what = "causal_conv_grad"
    ops, x, weight, bias, initial, resets, lengths, window, sizes = _conv_operands(
        what, x, weight, bias, initial, resets, lengths, activation, grad
    )
    grad = ops.array("grad", grad, x._shape)
    dx, d_weight, d_bias, d_initial = ops.backend.causal_conv_grad(grad, x, weight, bias, initial, resets, lengths, *sizes)
    return (
        ops.result(dx, x._shape),
        ops.result(d_weight, weight._shape),
        None if bias is None else ops.result(d_bias, bias._shape),
        None if initial is None else ops.result(d_initial, window),
    )


# ---- selective scan ----------------------------------------------------------------

_MOST_STATES = 256


def _scan_parameters(ops, channels, a_log, skip, delta_bias):
    a_log = ops.array("a_log", a_log)
    if len(a_log._shape) != 2 or a_log._shape[0] != channels:
        raise ValueError(f"{ops.what}: a_log must have shape ({channels}, states), got {a_log.shape}")
    states = a_log._shape[1]
    if not 1 <= states <= _MOST_STATES:
        raise ValueError(f"{ops.what}: a_log must have 1 to {_MOST_STATES} states, got {states}")
    return a_log, ops.optional("skip", skip, (channels,)), ops.optional("delta_bias", delta_bias, (channels,)), states


def _projections(ops, steps, channels, states, b, c):
    b = ops.array("b", b)
    if len(b._shape) != len(steps) + 2 or b._shape[:-2] != steps or b._shape[-1] != states:
        raise ValueError(f"{ops.what}: b must have shape {steps} and axes (groups, {states}), got {b.shape}")
    groups = b._shape[-2]
    if channels % groups if groups else channels:
        raise ValueError(f"{ops.what}: {groups} groups do not divide {channels} channels")
    if groups and not channels:
        raise ValueError(f"{ops.what}: {groups} groups without channels")
    return b, ops.array("c", c, b._shape), groups


def _scan_operands(what, x, delta, a_log, b, c, skip, gate, initial, delta_bias, resets, lengths, *others):
    ops, x, resets, lengths, lead, sizes = _sequence_operands(
        what, x, resets, lengths, delta, a_log, b, c, skip, gate, initial, delta_bias, *others
    )
    delta = ops.array("delta", delta, x._shape)
    a_log, skip, delta_bias, states = _scan_parameters(ops, sizes[2], a_log, skip, delta_bias)
    b, c, groups = _projections(ops, x._shape[:-1], sizes[2], states, b, c)
    gate = ops.optional("gate", gate, x._shape)
    whole = lead + (sizes[2], states)
    initial = ops.optional("initial", initial, whole)
    return ops, (x, delta, a_log, b, c, skip, gate, initial, delta_bias, resets, lengths), whole, sizes + (groups, states)


def selective_scan(x, delta, a_log, b, c, skip=None, gate=None, initial=None, *, delta_bias=None, resets=None, lengths=None):
    """A state space recurrence whose steps the inputs select: (y, last states).

    With ``dt = softplus(delta + delta_bias)`` each channel has ``states`` states
    ``h_t = exp(-dt exp(a_log)) h_{t-1} + dt x_t b_t`` and
    ``y_t = (sum c_t h_t + skip x_t) gate_t sigmoid(gate_t)``, without the last
    factor if ``gate`` is not given; ``exp(a_log)`` ends at the dtype's largest number.
    Shapes: x, delta, gate (..., time, channels);
    a_log (channels, states), of 1 to 256 states; b, c (..., time, groups, states),
    whose groups divide the channels; skip, delta_bias (channels,); ``initial``
    (..., channels, states), the states before the first step, zero if not
    given. Where ``resets`` (..., time) is true the states before that step count
    as zero, whatever they hold. Rows end after ``lengths`` (...) steps (all of
    them if not given, and at most): what is behind is not read, y is zero there
    and the last states (..., channels, states) are those of the row's last step.
    Equal calls give equal bits; a row's rounding may differ beside more or fewer rows.
    """
    ops, given, whole, sizes = _scan_operands("selective_scan", x, delta, a_log, b, c, skip, gate, initial, delta_bias, resets, lengths)
    y, last = ops.backend.selective_scan(*given, *sizes)
    return ops.result(y, given[0]._shape), ops.result(last, whole)


def selective_scan_step(x, delta, a_log, b, c, state, skip=None, gate=None, *, delta_bias=None):
    """One token: (y, new states) of x, delta, gate (..., channels) and b, c (..., groups, states), from ``state``."""
    what = "selective_scan_step"
    ops = _Operands(what, x, delta, a_log, b, c, state, skip, gate, delta_bias)
    x = ops.array("x", x)
    if not x._shape:
        raise ValueError(f"{what}: x must have axes (..., channels), got {x.shape}")
    lead, channels = x._shape[:-1], x._shape[-1]
    delta = ops.array("delta", delta, x._shape)
    a_log, skip, delta_bias, states = _scan_parameters(ops, channels, a_log, skip, delta_bias)
    b, c, groups = _projections(ops, lead, channels, states, b, c)
    gate = ops.optional("gate", gate, x._shape)
    state = ops.array("state", state, lead + (channels, states))
    y, last = ops.backend.selective_scan(
        x, delta, a_log, b, c, skip, gate, state, delta_bias, None, None, prod(lead), 1, channels, groups, states
    )
    return ops.result(y, x._shape), ops.result(last, state._shape)


class ScanGrads(NamedTuple):
    """Gradients of ``selective_scan``; None for what is not given."""

    x: object
    delta: object
    a_log: object
    b: object
    c: object
    skip: object
    gate: object
    delta_bias: object
    initial: object


def selective_scan_grad(grad, x, delta, a_log, b, c, skip=None, gate=None, initial=None, *, delta_bias=None, resets=None, lengths=None, grad_state=None):
    """Gradients (a ``ScanGrads``) of ``selective_scan`` whose y has the gradient ``grad`` and whose last
    states have ``grad_state`` (zero if not given).

    b and c get the sums over their group's channels, a_log, skip and
    delta_bias those over all steps. Equal calls give equal bits.
    """
    what = "selective_scan_grad"
    ops, given, whole, sizes = _scan_operands(
        what, x, delta, a_log, b, c, skip, gate, initial, delta_bias, resets, lengths, grad, grad_state
    )
    grad, grad_state = ops.array("grad", grad, given[0]._shape), ops.optional("grad_state", grad_state, whole)
    found = ops.backend.selective_scan_grad(grad, grad_state, *given, *sizes)
    like = given[:7] + (given[8], given[7])
    return ScanGrads(*(None if array is None else ops.result(data, array._shape) for data, array in zip(found, like)))


# ---- residual stream and norms -------------------------------------------------------


def _norm_operands(what, x, stream, weight, post_weight, gate, scale, eps, *others):
    ops = _Operands(what, x, stream, weight, post_weight, gate, *others)
    x = ops.array("x", x)
    if not x._shape or not x._shape[-1]:
        raise ValueError(f"{what}: x must have axes (..., channels), none of it empty, got {x.shape}")
    lead, channels = x._shape[:-1], x._shape[-1]
    weight = ops.array("weight", weight, (channels,))
    post_weight = ops.optional("post_weight", post_weight, (channels,))
    divide = 1
    if gate is not None:
        gate = ops.array("gate", gate)
        # Leading axes as x has them, then ones: a factor for `divide` neighbouring rows.
        whole = (1,) * (len(x._shape) - len(gate._shape)) + gate._shape
        kept = max((i + 1 for i, d in enumerate(whole[:-1]) if d != 1), default=0)
        if whole != lead[:kept] + (1,) * (len(lead) - kept) + (channels,):
            raise ValueError(f"{what}: gate must have x's channels, and x's leading axes up to one and 1 after it, got {gate.shape} for {x.shape}")
        divide = prod(lead[kept:])
    scale, eps = _number("scale", scale), _number("eps", eps, 0)
    if eps < _TINY[ops.dtype]:
        raise ValueError(f"eps must be positive, and at least {_TINY[ops.dtype]} for {ops.dtype}")
    return ops, x, weight, post_weight, gate, (prod(lead), channels, divide, scale, eps)


def residual_norm(x, residual, weight, *, post_weight=None, gate=None, scale=1.0, eps=1e-6):
    """The residual stream after a block, and the next block's normed input: (stream, normed).

    With ``rms(v) = v / sqrt(mean(v v) + eps)`` over the last axis, for x, the
    block's output, and the stream before it:
    ``stream = residual + scale gate rms(x) post_weight`` and
    ``normed = rms(stream) weight``. Without ``post_weight`` x itself takes the
    place of rms(x) post_weight; without ``gate`` it is one. ``gate`` has the
    channels, and any number of x's leading axes followed by axes of 1: one
    factor for each token and channel, each sequence and channel, or each channel.
    The mean of the squares is formed in the arrays' dtype: a row that it overflows
    (values past 1.8e19 in float32) has an rms(v) of zero.
    """
    what = "residual_norm"
    ops, x, weight, post_weight, gate, sizes = _norm_operands(what, x, residual, weight, post_weight, gate, scale, eps)
    residual = ops.array("residual", residual, x._shape)
    stream, normed = ops.backend.residual_norm(x, residual, weight, post_weight, gate, *sizes)
    return ops.result(stream, x._shape), ops.result(normed, x._shape)


def residual_norm_grad(grad_stream, grad_normed, x, stream, weight, *, post_weight=None, gate=None, scale=1.0, eps=1e-6):
    """Gradients (x, residual, weight, post_weight, gate) of ``residual_norm``, whose ``stream`` it found.

    ``grad_stream`` and ``grad_normed`` are the gradients of its two results.
    What is not given has None. Equal calls give equal bits.
    """
    what = "residual_norm_grad"
    ops, x, weight, post_weight, gate, sizes = _norm_operands(
        what, x, stream, weight, post_weight, gate, scale, eps, grad_stream, grad_normed
    )
    stream = ops.array("stream", stream, x._shape)
    grad_stream, grad_normed = ops.array("grad_stream", grad_stream, x._shape), ops.array("grad_normed", grad_normed, x._shape)
    found = ops.backend.residual_norm_grad(grad_stream, grad_normed, x, stream, weight, post_weight, gate, *sizes)
    like = (x, x, weight, post_weight, gate)
    return tuple(None if array is None else ops.result(data, array._shape) for data, array in zip(found, like))


# ---- losses from logits ----------------------------------------------------------


def _logits_operands(what, logits, *others):
    ops = _Operands(what, logits, *others)
    logits = ops.array("logits", logits)
    if not logits.ndim or not logits.shape[-1]:
        raise ValueError(f"{what}: logits must have axes (..., vocabulary), none of it empty, got {logits.shape}")
    return ops, logits, logits.shape[:-1]


def token_log_probs(logits, targets, *, mask=None):
    """``log softmax(logits)`` over the last axis at the integer ``targets``; zero where ``mask`` is false.

    Rows that the mask leaves out are not read, and their targets may be
    anything. Another target outside the vocabulary gives NaN. Equal calls give
    equal bits; a long row's rounding may differ beside more or fewer rows.
    """
    ops, logits, tokens = _logits_operands("token_log_probs", logits, targets, mask)
    targets = ops.array("targets", targets, tokens, _INDICES)
    mask = ops.optional("mask", mask, tokens, (_BOOL,))
    return ops.result(ops.backend.token_log_probs(logits, targets, mask), tokens)


def _policy(what, gradient, logits, actions, old_log_probs, advantages, reference_log_probs, mask, clip, kl_weight, count):
    ops, logits, tokens = _logits_operands(what, logits, actions, old_log_probs, advantages, reference_log_probs, mask)
    actions = ops.array("actions", actions, tokens, _INDICES)
    old_log_probs = ops.array("old_log_probs", old_log_probs, tokens)
    advantages = ops.broadcast("advantages", advantages, tokens)
    reference = ops.optional("reference_log_probs", reference_log_probs, tokens)
    mask = ops.optional("mask", mask, tokens, (_BOOL,))
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    low, high = _number("clip", low, 0, infinite=True), _number("clip", high, 0, infinite=True)
    kl_weight = _number("kl_weight", kl_weight, 0)
    if kl_weight and reference is None:
        raise ValueError(f"{what}: kl_weight needs reference_log_probs")
    if count is not None:
        count = _positive("count", count)
    loss, log_probs, d_logits = ops.backend.policy_loss(
        logits, actions, old_log_probs, advantages, reference if kl_weight else None, mask, low, high, kl_weight, count, gradient
    )
    found = ops.result(loss, ()), ops.result(log_probs, tokens)
    return found + (ops.result(d_logits, logits.shape),) if gradient else found


def policy_loss(logits, actions, old_log_probs, advantages, *, reference_log_probs=None, mask=None, clip=0.2, kl_weight=0.0, count=None):
    """Clipped policy loss of tokens with a KL term: (loss, log-probabilities of the actions).

    With the ratio ``r = exp(log_prob - old)`` a token's loss is
    ``-min(r A, clip(r, 1 - low, 1 + high) A) + kl_weight (exp(d) - d - 1)``, where
    ``d = reference - log_prob`` and ``clip`` is ``(low, high)`` or one number
    for both. The loss is the sum over the tokens that ``mask`` keeps, divided
    by their number, or by ``count`` (for batches in parts); zero where it keeps
    none. ``advantages`` broadcast to the tokens. Masked rows are not read.
    """
    return _policy("policy_loss", False, logits, actions, old_log_probs, advantages, reference_log_probs, mask, clip, kl_weight, count)


def policy_loss_grad(logits, actions, old_log_probs, advantages, *, reference_log_probs=None, mask=None, clip=0.2, kl_weight=0.0, count=None):
    """``policy_loss`` and the loss's gradient: (loss, log-probabilities, gradient of the logits).

    Where both sides of the minimum are equal the gradient is that of the
    ratio's side. Rows that the mask leaves out have gradient zero.
    """
    return _policy("policy_loss_grad", True, logits, actions, old_log_probs, advantages, reference_log_probs, mask, clip, kl_weight, count)


def _preference(what, gradient, logits, targets, reference_log_probs, mask, beta, smoothing):
    ops, logits, tokens = _logits_operands(what, logits, targets, reference_log_probs, mask)
    if len(tokens) != 3 or tokens[0] != 2:
        raise ValueError(f"{what}: logits must have axes (2, pairs, time, vocabulary), got {logits.shape}")
    targets = ops.array("targets", targets, tokens, _INDICES)
    reference = ops.array("reference_log_probs", reference_log_probs, tokens[:2])
    mask = ops.optional("mask", mask, tokens, (_BOOL,))
    beta, smoothing = _number("beta", beta), _number("smoothing", smoothing, 0)
    if smoothing > 1:
        raise ValueError(f"smoothing is out of range: {smoothing}")
    loss, sums, d_logits = ops.backend.preference_loss(logits, targets, reference, mask, beta, smoothing, gradient)
    found = ops.result(loss, ()), ops.result(sums, tokens[:2])
    return found + (ops.result(d_logits, logits.shape),) if gradient else found


def preference_loss(logits, targets, reference_log_probs, *, mask=None, beta=0.1, smoothing=0.0):
    """Loss of paired responses: (loss, log-probabilities of the responses, summed over the tokens that ``mask`` keeps).

    ``logits`` has axes (2, pairs, time, vocabulary): the chosen responses,
    then the rejected ones; ``reference_log_probs`` (2, pairs) are a reference
    model's sums. With ``m = beta ((chosen - its reference) - (rejected - its reference))``
    the loss is the mean over pairs of
    ``-(1 - smoothing) log sigmoid(m) - smoothing log sigmoid(-m)``, zero of no pairs.
    """
    return _preference("preference_loss", False, logits, targets, reference_log_probs, mask, beta, smoothing)


def preference_loss_grad(logits, targets, reference_log_probs, *, mask=None, beta=0.1, smoothing=0.0):
    """``preference_loss`` and its gradient: (loss, responses' log-probabilities, gradient of the logits)."""
    return _preference("preference_loss_grad", True, logits, targets, reference_log_probs, mask, beta, smoothing)


_MOST_LISTED = 1024


def _distillation(what, gradient, logits, indices, teacher_logits, teacher_rest, mask, temperature, count):
    ops, logits, tokens = _logits_operands(what, logits, indices, teacher_logits, teacher_rest, mask)
    indices = ops.array("indices", indices, dtypes=_INDICES)
    if not indices._shape or indices._shape[:-1] != tokens or not 1 <= indices._shape[-1] <= _MOST_LISTED:
        raise ValueError(f"{what}: indices must have shape {tokens} and an axis of 1 to {_MOST_LISTED} entries, got {indices.shape}")
    teacher_logits = ops.array("teacher_logits", teacher_logits, indices._shape)
    teacher_rest = ops.optional("teacher_rest", teacher_rest, tokens)
    mask = ops.optional("mask", mask, tokens, (_BOOL,))
    temperature = _positive("temperature", temperature)
    if temperature < _TINY[ops.dtype] or 1 / temperature < _TINY[ops.dtype]:
        raise ValueError(f"temperature is out of range: {temperature}")
    if count is not None:
        count = _positive("count", count)
    loss, losses, d_logits = ops.backend.distillation_loss(
        logits, indices, teacher_logits, teacher_rest, mask, temperature, count, gradient
    )
    found = ops.result(loss, ()), ops.result(losses, tokens)
    return found + (ops.result(d_logits, logits.shape),) if gradient else found


def distillation_loss(logits, indices, teacher_logits, teacher_rest=None, *, mask=None, temperature=1.0, count=None):
    """Divergence of the logits' softmax from a teacher known by its largest logits: (loss, losses of the tokens).

    ``teacher_logits`` (..., entries) stand at the vocabulary's ``indices`` (...,
    entries), 1 to 1024 of them. Both sides are divided by ``temperature``. The
    teacher's distribution p is the softmax of its list, q that of all logits,
    and a token's loss is ``sum p (log p - log q)`` over the list. With
    ``teacher_rest`` (...), the log-sum-exp of the teacher's other logits over the
    temperature, p has the rest of the vocabulary as one more class, whose q is
    the sum over all logits that the list does not name. An entry of -inf is
    none, and its index may be anything; another index outside the vocabulary
    gives NaN; an index that stands twice is two entries of the sum. The loss is
    the sum over the tokens that ``mask`` keeps, divided by their number or by
    ``count``; zero where it keeps none. Masked rows are not read and have
    losses of zero. Equal calls give equal bits.
    """
    return _distillation("distillation_loss", False, logits, indices, teacher_logits, teacher_rest, mask, temperature, count)


def distillation_loss_grad(logits, indices, teacher_logits, teacher_rest=None, *, mask=None, temperature=1.0, count=None):
    """``distillation_loss`` and its gradient: (loss, losses of the tokens, gradient of the logits)."""
    return _distillation("distillation_loss_grad", True, logits, indices, teacher_logits, teacher_rest, mask, temperature, count)


# ---- AdamW ---------------------------------------------------------------------


class AdamWState:
    """Moments of ``adamw`` for a list of tensors; made by ``adamw_state`` and by each step.

    ``steps``: steps taken. ``first``, ``second``: the moments as lists of
    arrays, one of each tensor's shape. ``state_bits``: 8, or None where the
    moments have the parameters' dtype. A state is a value: a step makes a new
    one and leaves it as it was.
    """

    def __init__(self, backend, dtype, shapes, state_bits, steps, data):
        self._backend, self._dtype, self._shapes, self._data = backend, dtype, shapes, data
        self.state_bits, self.steps = state_bits, steps

    def _moments(self, which):
        storages = self._backend.adamw_moments(self._data, which, self._shapes, self._dtype, self.state_bits)
        return _wrapped_list(storages, self._shapes, self._dtype, self._backend)

    @property
    def first(self):
        return self._moments(0)

    @property
    def second(self):
        return self._moments(1)

    def __repr__(self):
        return f"AdamWState(tensors={len(self._shapes)}, steps={self.steps}, state_bits={self.state_bits}, dtype={self._dtype})"


def _wrapped_list(storages, shapes, dtype, backend):
    arrays, new, kind = [], object.__new__, xp.ndarray
    for data, shape in zip(storages, shapes):  # _wrapped, without a call for each of many tensors
        array = new(kind)
        array._data, array._shape, array._dtype, array._backend = data, shape, dtype, backend
        arrays.append(array)
    return arrays


def _check_tensors(what, name, values, backend, dtype, shapes):
    """Refuse what is not a list of arrays of this backend, dtype and these shapes."""
    if type(values) in (list, tuple) and len(values) == len(shapes):
        try:  # of as many tensors none is left out where all shapes are found
            if [v._shape for v in values if v._backend is backend and v._dtype is dtype] == shapes:
                return
        except AttributeError:
            pass  # something in it is no array
    if not isinstance(values, (list, tuple)) or not all([isinstance(v, xp.ndarray) for v in values]):
        raise TypeError(f"{what}: {name} must be a list of arrays")
    for value in values:
        if value._backend is not backend:
            raise BackendMismatchError("Arrays belong to different backends/devices; use to_backend()")
        if value._dtype is not dtype and value._dtype != dtype:
            raise UnsupportedDtypeError(f"{what}: {name} must be {dtype}, got {value.dtype}")
    if [v._shape for v in values] != shapes:
        raise ValueError(f"{what}: the shapes of {name} do not match those of the state's {len(shapes)} tensors")


def adamw_state(params, *, state_bits=None, steps=0, first=None, second=None):
    """The state before the first step of ``adamw`` on ``params``, or one that is taken up again
    after ``steps`` steps with the moments ``first`` and ``second``.

    ``state_bits=8`` (float32 parameters only) keeps each moment in one byte an
    element with a float32 scale for every 256 elements of a tensor: sign, 3 exponent bits and
    4 bits of the first moment's share in the block's largest, 4 exponent bits
    and 4 bits of the second's root, each rounded to the nearest; a moment that
    is not finite makes its block NaN. A moment moves once its change passes
    half a step of its code.
    """
    what = "adamw_state"
    if isinstance(params, (list, tuple)) and not params:
        raise ValueError(f"{what}: no tensors")
    if not isinstance(params, (list, tuple)) or not isinstance(params[0], xp.ndarray):
        raise TypeError(f"{what}: params must be a list of arrays")
    backend, dtype = params[0]._backend, params[0]._dtype
    _refuse_capture(what, backend)
    if dtype not in _FLOATS:
        raise UnsupportedDtypeError(f"{what} requires float32 or float64, got {dtype}")
    shapes = [getattr(p, "_shape", None) for p in params]
    _check_tensors(what, "params", params, backend, dtype, shapes)
    if state_bits not in (None, 8):
        raise ValueError(f"state_bits must be None or 8, got {state_bits!r}")
    if state_bits == 8 and dtype != _FLOATS[0]:
        raise UnsupportedDtypeError("states of 8 bits belong to float32 parameters")
    steps = operator.index(steps)
    if steps < 0:
        raise ValueError("steps must not be negative")
    if (first is None) != (second is None):
        raise ValueError("first and second come together")
    for name, moments in (("first", first), ("second", second)):
        if moments is not None:
            _check_tensors(what, name, moments, backend, dtype, shapes)
    return AdamWState(backend, dtype, shapes, state_bits, steps, backend.adamw_load(first, second, shapes, dtype, state_bits))


def adamw(params, grads, state, *, learning_rate=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01):
    """One AdamW step over a list of tensors: (new params, new state).

    ``m = b1 m + (1 - b1) g``, ``v = b2 v + (1 - b2) g g`` and, in step t,
    ``p - learning_rate (weight_decay p + (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps))``.
    ``weight_decay`` is one number or one for each tensor. The new parameters
    share one allocation, which lives as long as any of them.
    """
    what = "adamw"
    if not isinstance(state, AdamWState):
        raise TypeError(f"{what}: state must come from adamw_state or a step")
    backend, dtype, shapes = state._backend, state._dtype, state._shapes
    _refuse_capture(what, backend)
    _check_tensors(what, "params", params, backend, dtype, shapes)
    _check_tensors(what, "grads", grads, backend, dtype, shapes)
    learning_rate = _number("learning_rate", learning_rate, 0)
    beta1, beta2 = (_number("betas", b, 0, 1) for b in betas)
    eps = _number("eps", eps, 0)
    if eps < _TINY[dtype]:
        raise ValueError(f"eps must be positive, and at least {_TINY[dtype]} for {dtype}")
    if type(weight_decay) is not float and np.ndim(weight_decay):
        decays = [_number("weight_decay", d, 0) for d in weight_decay]
        if len(decays) != len(shapes):
            raise ValueError(f"{what}: {len(decays)} values of weight_decay for {len(shapes)} tensors")
    else:
        decays = [_number("weight_decay", weight_decay, 0)] * len(shapes)
    steps = state.steps + 1
    # In 64 bits, once: the step size, the root's factor and each tensor's decay.
    scalars = (beta1, beta2, learning_rate / (1 - beta1**steps), 1 / math.sqrt(1 - beta2**steps), eps)
    decays = [learning_rate * d for d in decays]
    storages, data = backend.adamw_step(params, grads, state._data, shapes, dtype, state.state_bits, decays, scalars)
    return _wrapped_list(storages, shapes, dtype, backend), AdamWState(backend, dtype, shapes, state.state_bits, steps, data)
