"""The operators of ``nn`` on the hip backend: storage for the results and one
library call each. Arguments arrive checked (nn.py); None stands for an
operand that is not given."""

import ctypes
from math import prod

from . import _hip_lib as lib_


def _ptr(array):
    return None if array is None else array._data.ptr


def _run(backend, name, *args):
    with backend._guard:
        backend._call(name, *args)


def gated_recurrence(backend, x, gate, initial, resets, batch, time, channels, gates):
    h = backend.empty(x._shape, x._dtype)
    _run(
        backend, "hp_gated_recurrence", lib_.DTYPE_CODES[x._dtype], x._data.ptr, gate._data.ptr, _ptr(initial), _ptr(resets),
        h.ptr, batch, time, channels, gates,
    )
    return h


def gated_recurrence_grad(backend, grad, x, gate, h, initial, resets, batch, time, channels, gates):
    dx, d_gate = backend.empty(x._shape, x._dtype), backend.empty(gate._shape, x._dtype)
    d_initial = None
    if initial is not None:
        # Of no steps the states do not depend on it.
        d_initial = backend.empty(initial._shape, x._dtype) if time else backend.full(initial._shape, 0, x._dtype)
    _run(
        backend, "hp_gated_recurrence_grad", lib_.DTYPE_CODES[x._dtype], grad._data.ptr, x._data.ptr, gate._data.ptr,
        h._data.ptr, _ptr(initial), _ptr(resets), dx.ptr, d_gate.ptr, None if d_initial is None else d_initial.ptr,
        batch, time, channels, gates,
    )
    return dx, d_gate, d_initial


def _codes(logits, targets):
    return lib_.DTYPE_CODES[logits._dtype], lib_.DTYPE_CODES[targets._dtype]


def token_log_probs(backend, logits, targets, mask):
    log_probs = backend.empty(targets._shape, logits._dtype)
    _run(
        backend, "hp_token_log_probs", *_codes(logits, targets), logits._data.ptr, targets._data.ptr, _ptr(mask), log_probs.ptr,
        targets.size, logits._shape[-1],
    )
    return log_probs


def _period(shape, whole):
    """(divide, period) such that element (i // divide) % period of an array of
    `shape` stands at element i of it broadcast to `whole`; None where the axes
    that it has are not next to each other."""
    shape = (1,) * (len(whole) - len(shape)) + shape
    kept = [axis for axis, (own, d) in enumerate(zip(shape, whole)) if own == d != 1]
    if not kept:
        return 1, 1
    if any(whole[axis] != 1 for axis in range(kept[0], kept[-1]) if axis not in kept):
        return None
    return prod(whole[kept[-1] + 1 :]), prod(shape)


def _broadcast(backend, array, whole):
    """Storage of `array`, and how it repeats over `whole` (_period)."""
    if array._shape == whole:
        return array._data, 1, max(1, array.size)
    if whole and array._shape == whole[:-1] + (1,):  # one for each row, the usual one
        return array._data, max(1, whole[-1]), max(1, array.size)
    found = _period(array._shape, whole)
    if found is None and not prod(whole):
        found = 1, 1  # nothing is read
    if found is None:
        strides = [prod(array._shape[axis + 1 :]) if d != 1 else 0 for axis, d in enumerate(array._shape)]
        return backend.gather(array, whole, 0, (0,) * (len(whole) - len(strides)) + tuple(strides)), 1, prod(whole)
    return array._data, *(max(1, n) for n in found)


def policy_loss(backend, logits, actions, old, advantages, reference, mask, low, high, kl_weight, count, gradient):
    loss, log_probs = backend.empty((), logits._dtype), backend.empty(actions._shape, logits._dtype)
    grad = backend.empty(logits._shape, logits._dtype) if gradient else None
    gains, divide, period = _broadcast(backend, advantages, actions._shape)
    _run(
        backend, "hp_policy_loss", *_codes(logits, actions), logits._data.ptr, actions._data.ptr, old._data.ptr, gains.ptr,
        divide, period, _ptr(reference), _ptr(mask), loss.ptr, log_probs.ptr, None if grad is None else grad.ptr,
        actions.size, logits._shape[-1], low, high, kl_weight, count or 0.0,
    )
    return loss, log_probs, grad


def preference_loss(backend, logits, targets, reference, mask, beta, smoothing, gradient):
    loss, sums = backend.empty((), logits._dtype), backend.empty(reference._shape, logits._dtype)
    grad = backend.empty(logits._shape, logits._dtype) if gradient else None
    _, pairs, time = targets._shape
    _run(
        backend, "hp_preference_loss", *_codes(logits, targets), logits._data.ptr, targets._data.ptr, reference._data.ptr,
        _ptr(mask), loss.ptr, sums.ptr, None if grad is None else grad.ptr, pairs, time, logits._shape[-1], beta, smoothing,
    )
    return loss, sums, grad


# ---- AdamW ---------------------------------------------------------------------


class _Span:
    """Storage of one tensor inside a block that several share, which it keeps."""

    __slots__ = ("block", "offset")

    @property
    def ptr(self):
        start = self.block.ptr  # 0 once the backend is closed
        return start + self.offset if start else 0


class _Layout:
    """Places of tensors of one dtype within the arrays of a state (hp_adamw_layout)."""

    def __init__(self, backend, shapes, dtype, bits):
        self.code, self.bits, self.count = lib_.DTYPE_CODES[dtype], bits or 0, len(shapes)
        self.sizes = lib_.int64_array(prod(shape) for shape in shapes)
        offsets, elements, state_bytes = lib_.int64_array([0] * self.count), ctypes.c_int64(), ctypes.c_int64()
        status = backend._lib.hp_adamw_layout(
            self.code, self.bits, self.count, self.sizes, offsets, ctypes.byref(elements), ctypes.byref(state_bytes)
        )
        lib_.check(backend._lib, status, "hp_adamw_layout")
        self.offsets = [offset * dtype.itemsize for offset in offsets[: self.count]]
        self.elements, self.bytes = elements.value, elements.value * dtype.itemsize
        self.state_bytes = max(1, state_bytes.value)
        self.pointers, self.numbers = ctypes.c_void_p * self.count, ctypes.c_double * self.count

    def addresses(self, arrays):
        return self.pointers(*[a._data.ptr for a in arrays])

    def spans(self, block, start=0):
        spans, new = [], object.__new__
        for offset in self.offsets:
            span = new(_Span)
            span.block, span.offset = block, start + offset
            spans.append(span)
        return spans


class _State:
    __slots__ = ("layout", "block")

    def __init__(self, layout, block):
        self.layout, self.block = layout, block


def adamw_load(backend, first, second, shapes, dtype, bits):
    layout = _Layout(backend, shapes, dtype, bits)
    block = backend.block(layout.state_bytes)
    if first is None:
        _run(backend, "hp_fill", block.ptr, layout.state_bytes, 1, 0)
    else:
        _run(
            backend, "hp_adamw_load", layout.code, layout.bits, layout.count, layout.addresses(first), layout.addresses(second),
            layout.sizes, block.ptr,
        )
    return _State(layout, block)


def adamw_moments(backend, state, which, shapes, dtype, bits):
    layout = state.layout
    if not bits:
        return layout.spans(state.block, which * layout.bytes)
    values = backend.block(max(1, layout.bytes))
    _run(backend, "hp_adamw_values", layout.elements, state.block.ptr, which, values.ptr)
    return layout.spans(values)


def adamw_step(backend, params, grads, state, shapes, dtype, bits, decays, scalars):
    layout = state.layout
    block, new = backend.block(layout.state_bytes), backend.block(max(1, layout.bytes))
    _run(
        backend, "hp_adamw_step", layout.code, layout.bits, layout.count, layout.addresses(params), layout.addresses(grads),
        layout.sizes, layout.numbers(*decays), state.block.ptr, block.ptr, new.ptr, *scalars,
    )
    return layout.spans(new), _State(layout, block)
