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


# ---- losses from logits ----------------------------------------------------------
#
# Bounds are in units of rounding u of the operator's type. A row's sum of
# exponentials loses 50 u in its terms' own rounding and the sum's order (an
# exponential 4, a tree and chains of at most some tens of additions), and
# D = sum_j p_j |z_j - max| u from the subtractions; its logarithm and the
# differences add their own sizes.


class Row:
    """One row of logits and its target."""

    def __init__(self, logits, target):
        z = np.asarray(logits).astype(WIDE)
        top = z.max()
        terms = np.exp(z - top)
        total = terms.sum()
        self.p, self.target = terms / total, target
        self.distance = np.where(self.p > 0, np.abs(z - top), 0)
        self.total_units = 50 + (self.p * self.distance).sum()
        self.log_prob = z[target] - top - np.log(total)
        self.units = self.total_units + 3 * abs(np.log(total)) + 2 * abs(z[target] - top) + abs(self.log_prob)

    def grad(self, weight, weight_units):
        """weight (1[target] - p), and its bound for a weight that is off by weight_units."""
        one = np.zeros_like(self.p)
        one[self.target] = 1
        p_units = 6 + self.distance + self.total_units
        bound = weight_units * np.abs(one - self.p) + abs(weight) * (self.p * p_units + 2 * one)
        return weight * (one - self.p), bound


def token_log_probs(logits, targets, mask=None):
    """(values, bounds in units of rounding) over rows of logits (rows, vocabulary)."""
    values, units = np.zeros(len(logits), WIDE), np.zeros(len(logits), WIDE)
    for i in range(len(logits)):
        if mask is None or mask[i]:
            row = Row(logits[i], targets[i])
            values[i], units[i] = row.log_prob, row.units
    return values, units


def policy_loss(logits, actions, old, advantages, reference=None, mask=None, clip=(0.2, 0.2), kl_weight=0.0, count=None):
    """((loss, log_probs, gradient), their bounds, rows whose ratio is so near an end of the clip
    that rounding decides between the sides), over rows of logits."""
    old, advantages, reference = _wide(old, advantages, reference)
    n = len(logits)
    log_probs, units = np.zeros(n, WIDE), np.zeros(n, WIDE)
    grad, bounds = np.zeros(np.shape(logits), WIDE), np.zeros(np.shape(logits), WIDE)
    loss, loss_units, undecided = WIDE(0), WIDE(0), np.zeros(n, bool)
    kept = range(n) if mask is None else np.flatnonzero(mask)
    if count is None:
        count = max(1, len(kept))
    low, high = 1 - WIDE(clip[0]), 1 + WIDE(clip[1])
    for i in kept:
        row = Row(logits[i], actions[i])
        log_probs[i], units[i] = row.log_prob, row.units
        ratio = np.exp(row.log_prob - old[i])
        ratio_units = ratio * (row.units + abs(row.log_prob - old[i]) + 3)
        undecided[i] = min(abs(ratio - low), abs(ratio - high)) <= ratio_units * 2.0**-23 + 2.0**-22
        free, held = ratio * advantages[i], min(max(ratio, low), high) * advantages[i]
        stopped = free > held
        each, slope = -min(free, held), 0 if stopped else -free
        each_units = abs(advantages[i]) * ratio_units + 4 * abs(free)
        if reference is not None and kl_weight:
            apart = reference[i] - row.log_prob
            apart_units = row.units + abs(apart)
            each = each + kl_weight * (np.expm1(apart) - apart)
            slope = slope - kl_weight * np.expm1(apart)
            each_units += kl_weight * ((np.exp(apart) + 1) * apart_units + 4 * abs(np.expm1(apart)) + 2 * abs(apart))
        loss, loss_units = loss + each, loss_units + each_units + abs(each)
        grad[i], bounds[i] = row.grad(slope / count, (each_units + 4 * abs(slope)) / count)
    return (loss / count, log_probs, grad), (loss_units / count, units, bounds), undecided


def preference_loss(logits, targets, reference, mask=None, beta=0.1, smoothing=0.0):
    """((loss, sums, gradient), their bounds) of logits (2, pairs, time, vocabulary)."""
    _, pairs, time = np.shape(targets)
    (reference,) = _wide(reference)
    rows, sums, units = {}, np.zeros((2, pairs), WIDE), np.zeros((2, pairs), WIDE)
    for at in np.ndindex(2, pairs, time):
        if mask is None or mask[at]:
            rows[at] = row = Row(logits[at], targets[at])
            sums[at[:2]] += row.log_prob
            # Twenty additions deep in float, or one rounding of a double sum.
            units[at[:2]] += row.units + 20 * abs(row.log_prob)
    margin = WIDE(beta) * ((sums[0] - reference[0]) - (sums[1] - reference[1]))
    margin_units = abs(beta) * (units.sum(0) + 2 * np.abs(sums).sum(0) + 2 * np.abs(reference).sum(0)) + 4 * np.abs(margin)
    losses = (1 - smoothing) * np.log1p(np.exp(-margin)) + smoothing * np.log1p(np.exp(margin))
    loss_units = margin_units + 4 * (np.abs(margin) + 1)
    n = max(1, pairs)
    slope = beta * (smoothing * sigmoid(margin) - (1 - smoothing) * sigmoid(-margin)) / n
    slope_units = abs(beta) * (margin_units + 8) / n
    grad, bounds = np.zeros(np.shape(logits), WIDE), np.zeros(np.shape(logits), WIDE)
    for at, row in rows.items():
        grad[at], bounds[at] = row.grad(slope[at[1]] * (1 if at[0] == 0 else -1), slope_units[at[1]])
    return (losses.sum() / n, sums, grad), (loss_units.sum() / n, units + 4 * np.abs(sums), bounds)


# ---- AdamW ---------------------------------------------------------------------

BLOCK = 256


def adamw(p, g, m, v, steps, learning_rate, betas, eps, weight_decay):
    """((p', m', v'), their bounds in units of rounding) of one tensor in its step `steps`, as the definition has it."""
    p, g, m, v = _wide(p, g, m, v)
    b1, b2, rate, decay = (WIDE(x) for x in (*betas, learning_rate, weight_decay))
    # Constants, products and a sum: one rounding each.
    m_units, v_units = 4 * (np.abs(b1 * m) + np.abs((1 - b1) * g)), 5 * (np.abs(b2 * v) + (1 - b2) * g * g)
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    size = np.sqrt(v / (1 - b2**steps)) + eps
    move = rate * (m / (1 - b1**steps)) / size
    # The moment's own error, the root's (half of v's, which only sums terms >= 0), and some ten further roundings.
    p_units = rate / (1 - b1**steps) * m_units / size + (5 + 10) * np.abs(move) + 4 * np.abs(rate * decay * p)
    p = p - (rate * decay * p + move)
    return (p, m, v), (p_units + np.abs(p), m_units, v_units)


def _grid(codes, low):
    return np.array([c * 2.0**-low if c < 16 else (16 + c % 16) * 2.0 ** (c // 16 - 1 - low) for c in range(codes + 1)])


def _nearest(values, codes, low, positive):
    """float32 values >= 0 by the codes' shares of their block's largest; ties between codes go to the even one."""
    grid = _grid(codes, low)
    held = np.empty_like(values)
    for start in range(0, len(values), BLOCK):
        block = values[start : start + BLOCK]
        top = block.max()
        if not np.isfinite(top):
            held[start : start + BLOCK] = np.nan
            continue
        share = (block / top).astype(np.float64) if top > 0 else np.zeros(len(block))
        above = np.clip(np.searchsorted(grid, share), 1, codes)
        lower, upper = share - grid[above - 1], grid[above] - share
        code = np.where((upper < lower) | ((upper == lower) & (above % 2 == 0)), above, above - 1)
        if positive:
            code = np.where(block > 0, np.maximum(code, 1), code)
        held[start : start + BLOCK] = grid[code].astype(np.float32) * top
    return held


def held_first(m):
    """What a float32 first moment stands for in 8 bits."""
    flat = np.asarray(m, np.float32).reshape(-1)
    held = _nearest(np.abs(flat), 112, 10, False)
    return np.where(np.signbit(flat), -held, held).reshape(np.shape(m))


def held_second(v):
    flat = np.asarray(v, np.float32).reshape(-1)
    return np.square(_nearest(np.sqrt(flat), 240, 18, True)).reshape(np.shape(v))
