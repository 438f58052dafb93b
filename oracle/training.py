"""Plain forms of the training operators, in extended precision on the host.

Written from the definitions, one step or one row at a time, without the
package's own code. Beside each value stands the size of the terms that its
float computation rounds, so that tests can bound errors by what a computation
in the operator's precision has to lose.
"""

import numpy as np

WIDE = np.longdouble


def _wide(*arrays):
    return [None if a is None else np.asarray(a).astype(WIDE) for a in arrays]


def sigmoid(g):
    return 1 / (1 + np.exp(-g))


def _gate_columns(gate, channels):
    """(a, 1 - a) per channel of gates (batch, time, gates)."""
    width = channels // gate.shape[-1] if gate.shape[-1] else 1
    with np.errstate(over="ignore"):
        return np.repeat(sigmoid(gate), width, -1), np.repeat(sigmoid(-gate), width, -1)


def recurrence(x, gate, initial=None, resets=None):
    """States of (batch, time, channels), and the size of what each rounds: h_t sums terms of |a h| + |(1 - a) x|
    here and in every step before, each carried by the gates since."""
    x, gate, initial = _wide(x, gate, initial)
    batch, time, channels = x.shape
    a, take = _gate_columns(gate, channels)
    state = np.zeros((batch, channels), WIDE) if initial is None else initial
    size = np.zeros_like(state)
    h, sizes = np.empty_like(x), np.empty_like(x)
    for t in range(time):
        if resets is not None:
            state = np.where(resets[:, t, None], 0, state)
            size = np.where(resets[:, t, None], 0, size)
        size = a[:, t] * (size + np.abs(state)) + np.abs(take[:, t] * x[:, t])
        state = a[:, t] * state + take[:, t] * x[:, t]
        h[:, t], sizes[:, t] = state, size
    return h, sizes


def recurrence_grad(grad, x, gate, h, initial=None, resets=None):
    """(dx, dgate, dinitial) and the sizes of what each rounds."""
    grad, x, gate, h, initial = _wide(grad, x, gate, h, initial)
    batch, time, channels = x.shape
    a, take = _gate_columns(gate, channels)
    width = channels // gate.shape[-1] if gate.shape[-1] else 1
    carried, size = np.zeros((batch, channels), WIDE), np.zeros((batch, channels), WIDE)
    dx, dx_size = np.empty_like(x), np.empty_like(x)
    d_gate, gate_size = np.empty_like(gate), np.empty_like(gate)
    for t in reversed(range(time)):
        before = h[:, t - 1] if t else (np.zeros_like(carried) if initial is None else initial)
        if resets is not None:
            before = np.where(resets[:, t, None], 0, before)
        slope = grad[:, t] + carried
        size = size + np.abs(grad[:, t]) + np.abs(carried)
        dx[:, t], dx_size[:, t] = slope * take[:, t], size * take[:, t]
        share = slope * (before - x[:, t]) * a[:, t] * take[:, t]
        share_size = size * (np.abs(before) + np.abs(x[:, t])) * a[:, t] * take[:, t]
        d_gate[:, t] = share.reshape(d_gate[:, t].shape + (width,)).sum(-1)
        gate_size[:, t] = share_size.reshape(d_gate[:, t].shape + (width,)).sum(-1) * (1 + np.log2(max(2, width)))
        carried, size = a[:, t] * slope, a[:, t] * size
        if resets is not None:
            carried, size = (np.where(resets[:, t, None], 0, v) for v in (carried, size))
    return (dx, d_gate, carried), (dx_size, gate_size, size)
