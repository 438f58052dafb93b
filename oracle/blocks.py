"""Plain forms of the operators of a state space block and of its loss, in extended precision on the host.

Written from the definitions, without the package's own code, over numbers that
carry a running bound of what a computation in the operator's precision loses:
every operation adds its own rounding to what its operands are off by already.
"""

import numpy as np

from .training import WIDE, Row, sigmoid


class Number:
    """Values in extended precision, and how many units of rounding each may be off by (absolute)."""

    __slots__ = ("value", "units")

    def __init__(self, value, units=0):
        self.value = np.asarray(value).astype(WIDE)
        self.units = np.broadcast_to(np.asarray(units, WIDE), self.value.shape)

    def __getitem__(self, at):
        return Number(self.value[at], self.units[at])

    def __setitem__(self, at, other):
        self.units = self.units if self.units.flags.writeable else self.units.copy()
        self.value[at], self.units[at] = other.value, other.units

    def __add__(self, other):
        other = _number(other)
        # As large as its parts: sums may be formed in any order.
        return Number(self.value + other.value, self.units + other.units + np.abs(self.value) + np.abs(other.value))

    def __neg__(self):
        return Number(-self.value, self.units)

    def __sub__(self, other):
        return self + -_number(other)

    def __mul__(self, other):
        other = _number(other)
        value = self.value * other.value
        return Number(value, np.abs(self.value) * other.units + np.abs(other.value) * self.units + np.abs(value))

    __radd__, __rmul__ = __add__, __mul__

    def sum(self, axis):
        """A sum in any order, of trees and of chains of up to 64."""
        total = np.abs(self.value).sum(axis)
        return Number(self.value.sum(axis), self.units.sum(axis) + 64 * total)

    def map(self, function, slope, own):
        """function(value), whose derivative is at most `slope` in size, computed within `own` units of its value."""
        value = function(self.value)
        return Number(value, np.abs(slope) * self.units + own * np.abs(value))

    def where(self, condition, other=0.0):
        other = _number(other)
        return Number(np.where(condition, self.value, other.value), np.where(condition, self.units, other.units))

    def reshape(self, *shape):
        return Number(self.value.reshape(*shape), self.units.reshape(*shape))

    def repeat(self, times, axis):
        return Number(np.repeat(self.value, times, axis), np.repeat(self.units, times, axis))


def _number(value):
    return value if isinstance(value, Number) else Number(value)


def exp(v):
    value = np.exp(v.value)
    return Number(value, value * v.units + (4 + 2 * np.abs(v.value)) * value)


def silu_parts(v):
    """silu and its derivative."""
    s, r = sigmoid(v.value), sigmoid(-v.value)
    silu = Number(v.value * s, 1.1 * v.units + 8 * np.abs(v.value * s))
    slope = s * (1 + v.value * r)
    return silu, Number(slope, 0.5 * v.units + 10 * s * (1 + np.abs(v.value) * r))


def _softplus(v):
    value = np.maximum(v.value, 0) + np.log1p(np.exp(-np.abs(v.value)))
    # An exponential of -|v|, whose argument's rounding counts |v| times, a logarithm, a sum.
    return Number(value, sigmoid(v.value) * v.units + (12 + 2 * np.minimum(np.abs(v.value), 100)) * value)


def _ends(lengths, batch, time):
    return np.full(batch, time) if lengths is None else np.clip(np.asarray(lengths), 0, time)


# ---- causal convolution ----------------------------------------------------------


def _seen(whole, resets, taps, t, k):
    """What step t sees as tap k of (batch, taps - 1 + time, channels)."""
    seen = whole[:, t + k]
    if resets is None:
        return seen, np.ones(len(whole), bool)
    since = max(0, t - (taps - 1) + k + 1)  # a reset at one of these steps hides it
    visible = ~resets[:, since : t + 1].any(1) if k < taps - 1 else np.ones(len(whole), bool)
    return np.where(visible[:, None], seen, 0), visible


def causal_conv(x, weight, bias=None, initial=None, resets=None, lengths=None, activation=None, grad=None):
    """(y, last inputs), or with `grad` the gradients (x, weight, bias, initial), as Numbers."""
    batch, time, channels = x.shape
    taps = weight.shape[1]
    ends = _ends(lengths, batch, time)
    before = np.zeros((batch, taps - 1, channels), x.dtype) if initial is None else initial
    x = np.where((np.arange(time) < ends[:, None])[..., None], x, 0)
    whole = np.concatenate([before, x], 1)
    weight = Number(weight)
    y = Number(np.zeros(x.shape))
    d_whole, d_weight = Number(np.zeros(whole.shape)), Number(np.zeros(weight.value.shape))
    d_bias = Number(np.zeros(channels))
    for t in range(time):
        on = (t < ends)[:, None]
        pre = Number(np.zeros((batch, channels))) if bias is None else Number(np.broadcast_to(bias, (batch, channels)))
        for k in range(taps):
            pre = pre + weight[:, k] * _seen(whole, resets, taps, t, k)[0]
        value, slope = silu_parts(pre) if activation else (pre, Number(np.ones_like(pre.value)))
        y[:, t] = value.where(on)
        if grad is None:
            continue
        d = (slope * np.where(on, grad[:, t], 0)).where(on)
        d_bias = d_bias + d.sum(0)
        for k in range(taps):
            seen, visible = _seen(whole, resets, taps, t, k)
            d_whole[:, t + k] = d_whole[:, t + k] + (d * weight[:, k]).where(visible[:, None])
            d_weight[:, k] = d_weight[:, k] + (d * seen).sum(0)
    if grad is not None:
        return d_whole[:, taps - 1 :], d_weight, d_bias, d_whole[:, : taps - 1]
    last = np.zeros(before.shape, WIDE)
    for row in range(batch):
        for k in range(taps - 1):
            at = ends[row] - (taps - 1) + k  # a step, or below zero a carried input
            if resets is None or not resets[row, max(0, at + 1) : ends[row]].any():
                last[row, k] = whole[row, ends[row] + k]
    return y, last


# ---- selective scan ----------------------------------------------------------------


def selective_scan(x, delta, a_log, b, c, skip=None, gate=None, initial=None, delta_bias=None, resets=None, lengths=None,
                   grad=None, grad_state=None):
    """(y, last states), or with `grad` the gradients in the order of nn.ScanGrads, as Numbers."""
    batch, time, channels = x.shape
    groups, states = b.shape[2:]
    width = channels // groups if groups else 1
    ends = _ends(lengths, batch, time)
    inside = np.arange(time) < ends[:, None]

    def kept(v):
        return None if v is None else np.where(inside.reshape(inside.shape + (1,) * (v.ndim - 2)), v, 0)

    x, delta, b, c, gate, grad = (kept(v) for v in (x, delta, b, c, gate, grad))
    resets = np.zeros((batch, time), bool) if resets is None else resets
    rates = exp(Number(a_log))
    raw = Number(delta) if delta_bias is None else Number(delta) + delta_bias
    dt = _softplus(raw)

    def wide(v):
        return np.repeat(v, width, axis=1)

    state = Number(np.zeros((batch, channels, states)) if initial is None else initial)
    plain = Number(np.zeros(x.shape))
    befores, decays, afters = [], [], []
    for t in range(time):
        on = inside[:, t, None, None]
        before = state.where(~resets[:, t, None, None])
        decay = exp(-(dt[:, t][..., None] * rates))
        after = decay * before + (dt[:, t] * x[:, t])[..., None] * wide(b[:, t])
        # A run's decays are also composed from sums of dt: as many units again.
        after.units = after.units + 4 * np.abs(decay.value * before.value)
        y = (after * wide(c[:, t])).sum(-1)
        plain[:, t] = (y if skip is None else y + Number(skip) * x[:, t]).where(on[..., 0])
        state = after.where(on, state)
        befores.append(before), decays.append(decay), afters.append(after)
    silu = slope = None
    if gate is not None:
        silu, slope = silu_parts(Number(gate))
    if grad is None:
        return (plain if gate is None else plain * silu), state
    g = Number(grad) if gate is None else silu * grad
    lam = Number(np.zeros((batch, channels, states)) if grad_state is None else grad_state)
    dx, d_dt = Number(np.zeros(x.shape)), Number(np.zeros(x.shape))
    d_b, d_c = Number(np.zeros(b.shape)), Number(np.zeros(c.shape))
    d_rates = Number(np.zeros((channels, states)))

    def narrow(v):
        return v.reshape(batch, groups, width, states).sum(2)

    for t in reversed(range(time)):
        on = inside[:, t, None, None]
        bt, ct = wide(b[:, t]), wide(c[:, t])
        here = lam + g[:, t][..., None] * ct
        along, share = (here * bt).sum(-1), here * (decays[t] * befores[t])
        if groups:
            d_c[:, t] = narrow(g[:, t][..., None] * afters[t]).where(on)
            d_b[:, t] = narrow((dt[:, t] * x[:, t])[..., None] * here).where(on)
        part = along * dt[:, t]
        dx[:, t] = (part if skip is None else part + g[:, t] * skip).where(on[..., 0])
        d_dt[:, t] = (along * x[:, t] - (share * rates).sum(-1)).where(on[..., 0])
        d_rates = _gather(d_rates, -(share * dt[:, t][..., None]).where(on).sum(0))
        passed = (decays[t] * here).where(~resets[:, t, None, None])
        passed.units = passed.units + 4 * np.abs(passed.value)
        lam = passed.where(on, lam)
    d_delta = d_dt * raw.map(sigmoid, 0.25, 6)
    d_bias = d_delta.reshape(batch * time, channels).sum(0)
    d_skip = (g * x).reshape(batch * time, channels).sum(0)
    d_gate = None if gate is None else plain * grad * slope
    return dx, d_delta, d_rates * rates, d_b, d_c, d_skip, d_gate, d_bias, lam


def _gather(total, part):
    """A further term of a sum that is formed in trees, or in chains of up to 64."""
    return Number(total.value + part.value, total.units + part.units + 64 * np.abs(part.value))


# ---- residual stream and norms -------------------------------------------------------


def _unit(v, eps):
    """(v / rms(v), 1 / rms(v)) over the last axis."""
    n = v.value.shape[-1]
    square = (v * v).sum(-1) * (WIDE(1) / n) + WIDE(eps)
    inverse = Number(1 / np.sqrt(square.value), 0.5 * square.units / square.value**1.5 + 4 / np.sqrt(square.value))
    return v * inverse[..., None], inverse[..., None]


def _factor(gate, scale, rows, channels, divide):
    if gate is None:
        return Number(np.full((rows, channels), WIDE(scale)), abs(scale))
    return Number(np.repeat(np.asarray(gate).reshape(-1, channels), divide, axis=0)) * Number(WIDE(scale), abs(scale))


def residual_norm(x, residual, weight, post_weight=None, gate=None, divide=1, scale=1.0, eps=1e-6):
    """(stream, normed) of rows, as Numbers."""
    rows, channels = x.shape
    y = Number(x) if post_weight is None else _unit(Number(x), eps)[0] * post_weight
    stream = Number(residual) + _factor(gate, scale, rows, channels, divide) * y
    return stream, _unit(stream, eps)[0] * weight


def residual_norm_grad(grad_stream, grad_normed, x, stream, weight, post_weight=None, gate=None, divide=1, scale=1.0, eps=1e-6):
    """Gradients (x, residual, weight, post_weight, gate) of rows, as Numbers."""
    rows, channels = x.shape
    factor = _factor(gate, scale, rows, channels, divide)
    dn = Number(grad_normed)
    unit, outer = _unit(Number(stream), eps)
    through = dn * weight
    d = Number(grad_stream) + outer * (through - unit * ((through * unit).sum(-1) * (WIDE(1) / channels))[..., None])
    d_weight = (dn * unit).sum(0)
    dx, d_post, y = d * factor, None, Number(x)
    if post_weight is not None:
        unit, inner = _unit(Number(x), eps)
        d_post, through, y = (dx * unit).sum(0), dx * post_weight, unit * post_weight
        dx = inner * (through - unit * ((through * unit).sum(-1) * (WIDE(1) / channels))[..., None])
    d_gate = None if gate is None else (d * y * Number(WIDE(scale), abs(scale))).reshape(-1, divide, channels).sum(1)
    return dx, d, d_weight, d_post, d_gate


# ---- distillation ----------------------------------------------------------------


def distillation_loss(logits, indices, teacher, rest=None, mask=None, temperature=1.0, count=None):
    """((loss, losses, gradient), their bounds in units of rounding) over rows of logits."""
    n, vocab = logits.shape
    t = WIDE(temperature)
    losses, units = np.zeros(n, WIDE), np.zeros(n, WIDE)
    grad, bounds = np.zeros((n, vocab), WIDE), np.zeros((n, vocab), WIDE)
    kept = range(n) if mask is None else np.flatnonzero(mask)
    count = max(1, len(kept)) if count is None else WIDE(count)
    for i in kept:
        given = teacher[i].astype(WIDE) / t
        if rest is not None:
            given = np.append(given, rest[i].astype(WIDE))
        p = np.exp(given - given.max())
        p /= p.sum()
        # exp(x) of an x that is rounded to the type is off by |x| units besides the exponential's 4; the sum by as
        # many on the mean, and by its own 50; the quotient by 2.
        far = np.where(p > 0, np.abs(given - given.max()), 0)
        p_units = p * (56 + far + (p * far).sum())
        row = Row(logits[i].astype(WIDE) / t, 0)  # its shares of the vocabulary, and what they lose
        # Dividing by the temperature rounds every distance once more, and its inverse too.
        q, q_units = row.p, row.p * (8 + 3 * row.distance + 2 * row.total_units)
        named = indices[i].astype(np.int64)
        live = p[: len(named)] > 0
        unlisted = np.ones(vocab, bool)
        unlisted[named[live]] = False
        ahead = np.where(live, named, 0)
        log_q = (logits[i].astype(WIDE)[ahead] - logits[i].max()) / t - np.log(np.exp((logits[i].astype(WIDE) - logits[i].max()) / t).sum())
        terms, sizes = p[: len(named)].copy(), np.zeros(len(named), WIDE)
        with np.errstate(all="ignore"):
            log_p = np.log(p)
            terms = np.where(live, p[: len(named)] * (log_p[: len(named)] - log_q), 0)
            sizes = np.where(live, p[: len(named)] * (2 * row.total_units + 4) + p_units[: len(named)] * np.abs(log_p[: len(named)] - log_q), 0)
            sizes = np.where(np.isfinite(sizes), sizes, 0)
        losses[i], units[i] = terms.sum(), sizes.sum() + np.abs(terms).sum()
        outside = q.copy()
        out_units = q_units.copy()
        if rest is not None and p[-1] > 0:
            mass = q[unlisted].sum()
            mass_units = q_units[unlisted].sum() + 50 * mass
            losses[i] += p[-1] * (log_p[-1] - np.log(mass))
            units[i] += p[-1] * (mass_units / mass + 2 * row.total_units + 8) + p_units[-1] * np.abs(log_p[-1] - np.log(mass))
            outside = q - p[-1] * q / mass
            out_units = q_units + p[-1] * (q_units / mass + q * mass_units / mass**2 + 4 * q / mass) + p_units[-1] * q / mass
        grad[i] = np.where(unlisted, outside, q)
        bounds[i] = np.where(unlisted, out_units, q_units)
        np.subtract.at(grad[i], named[live], p[: len(named)][live])
        np.add.at(bounds[i], named[live], (p_units + p)[: len(named)][live])
        grad[i], bounds[i] = grad[i] / (t * count), (bounds[i] + 3 * np.abs(grad[i])) / (t * count)
    return (losses.sum() / count, losses, grad), ((units.sum() + 4 * np.abs(losses).sum()) / count, units + np.abs(losses), bounds)
