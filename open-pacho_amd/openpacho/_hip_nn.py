"""The operators of ``nn`` on the hip backend: storage for the results and one
library call each. Arguments arrive checked (nn.py); None stands for an
operand that is not given."""

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
