"""The operators of ``nn`` on the hip backend: storage for the results and one
library call each. Arguments arrive checked (nn.py); None stands for an
operand that is not given."""

import ctypes
from math import prod

from . import _hip_lib as lib_


def _ptr(array):
    return None if array is None else array._data.ptr


def gated_recurrence(backend, x, gate, initial, resets, batch, time, channels, gates):
    h = backend.empty(x.shape, x.dtype)
    with backend._active():
        backend._call(
            "hp_gated_recurrence", lib_.DTYPE_CODES[x.dtype], _ptr(x), _ptr(gate), _ptr(initial), _ptr(resets), h.ptr,
            batch, time, channels, gates,
        )
    return h


def gated_recurrence_grad(backend, grad, x, gate, h, initial, resets, batch, time, channels, gates):
    dx, d_gate = backend.empty(x.shape, x.dtype), backend.empty(gate.shape, gate.dtype)
    d_initial = None
    if initial is not None:
        # Of no steps the state does not depend on it.
        d_initial = backend.empty(initial.shape, x.dtype) if time else backend.full(initial.shape, 0, x.dtype)
    with backend._active():
        backend._call(
            "hp_gated_recurrence_grad", lib_.DTYPE_CODES[x.dtype], _ptr(grad), _ptr(x), _ptr(gate), _ptr(h), _ptr(initial),
            _ptr(resets), dx.ptr, d_gate.ptr, None if d_initial is None else d_initial.ptr, batch, time, channels, gates,
        )
    return dx, d_gate, d_initial


def _codes(logits, targets):
    return lib_.DTYPE_CODES[logits.dtype], lib_.DTYPE_CODES[targets.dtype]


def token_log_probs(backend, logits, targets, mask):
    log_probs = backend.empty(targets.shape, logits.dtype)
    with backend._active():
        backend._call(
            "hp_token_log_probs", *_codes(logits, targets), _ptr(logits), _ptr(targets), _ptr(mask), log_probs.ptr,
            targets.size, logits.shape[-1],
        )
    return log_probs


def policy_loss(backend, logits, actions, old, advantages, reference, mask, low, high, kl_weight, count, gradient):
    loss, log_probs = backend.empty((), logits.dtype), backend.empty(actions.shape, logits.dtype)
    grad = backend.empty(logits.shape, logits.dtype) if gradient else None
    with backend._active():
        backend._call(
            "hp_policy_loss", *_codes(logits, actions), _ptr(logits), _ptr(actions), _ptr(old), _ptr(advantages),
            _ptr(reference), _ptr(mask), loss.ptr, log_probs.ptr, None if grad is None else grad.ptr, actions.size,
            logits.shape[-1], low, high, kl_weight, count or 0.0,
        )
    return loss, log_probs, grad


def preference_loss(backend, logits, targets, reference, mask, beta, smoothing, gradient):
    loss, sums = backend.empty((), logits.dtype), backend.empty(reference.shape, logits.dtype)
    grad = backend.empty(logits.shape, logits.dtype) if gradient else None
    _, pairs, time = targets.shape
    with backend._active():
        backend._call(
            "hp_preference_loss", *_codes(logits, targets), _ptr(logits), _ptr(targets), _ptr(reference), _ptr(mask),
            loss.ptr, sums.ptr, None if grad is None else grad.ptr, pairs, time, logits.shape[-1], beta, smoothing,
        )
    return loss, sums, grad


# ---- AdamW ---------------------------------------------------------------------


class _Span:
    """Storage of one tensor inside a block that several share, which it keeps."""

    __slots__ = ("block", "offset")

    def __init__(self, block, offset):
        self.block, self.offset = block, offset

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
        return [_Span(block, start + offset) for offset in self.offsets]


class _State:
    __slots__ = ("layout", "block")

    def __init__(self, layout, block):
        self.layout, self.block = layout, block


def adamw_load(backend, first, second, shapes, dtype, bits):
    layout = _Layout(backend, shapes, dtype, bits)
    block = backend.block(layout.state_bytes)
    with backend._active():
        if first is None:
            backend._call("hp_fill", block.ptr, layout.state_bytes, 1, 0)
        else:
            backend._call(
                "hp_adamw_load", layout.code, layout.bits, layout.count, layout.addresses(first), layout.addresses(second),
                layout.sizes, block.ptr,
            )
    return _State(layout, block)


def adamw_moments(backend, state, which, shapes, dtype, bits):
    layout = state.layout
    if not bits:
        return layout.spans(state.block, which * layout.bytes)
    values = backend.block(max(1, layout.bytes))
    with backend._active():
        backend._call("hp_adamw_values", layout.elements, state.block.ptr, which, values.ptr)
    return layout.spans(values)


def adamw_step(backend, params, grads, state, shapes, dtype, bits, decays, scalars):
    layout = state.layout
    block, new = backend.block(layout.state_bytes), backend.block(max(1, layout.bytes))
    with backend._active():
        backend._call(
            "hp_adamw_step", layout.code, layout.bits, layout.count, layout.addresses(params), layout.addresses(grads),
            layout.sizes, layout.numbers(*decays), state.block.ptr, block.ptr, new.ptr, *scalars,
        )
    return layout.spans(new), _State(layout, block)
