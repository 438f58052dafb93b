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
