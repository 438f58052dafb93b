"""Host (NumPy backend) forms of the operators of ``nn``, in the arrays' dtype.

The mathematics stands at the functions of ``nn.py``; arrays come in and go
out as the NumPy backend's flat storage.
"""

import numpy as np

BLOCK = 256  # elements of a tensor that share the scale of an 8-bit moment
# Codes of the moments' shares of their block's largest, (codes, bits of the
# smallest): 16 steps an octave, the lowest 16 steps evenly down to zero.
FIRST, SECOND = (112, 10), (240, 18)


def _view(array):
    return None if array is None else array._data.reshape(array.shape)


# ---- gated recurrence ----------------------------------------------------------


def _gates(gate, width):
    """sigmoid(gate) and 1 - sigmoid(gate) of every channel, each to full precision."""
    small = np.exp(-np.abs(gate))
    high, low = 1 / (1 + small), small / (1 + small)
    keep, take = np.where(gate >= 0, high, low), np.where(gate >= 0, low, high)
    return np.repeat(keep, width, axis=-1), np.repeat(take, width, axis=-1)


def _axes(x, gate, initial, resets, batch, time, channels, gates):
    x, gate = _view(x).reshape(batch, time, channels), _view(gate).reshape(batch, time, gates)
    initial = np.zeros((batch, channels), x.dtype) if initial is None else _view(initial).reshape(batch, channels)
    resets = np.zeros((batch, time), bool) if resets is None else _view(resets).reshape(batch, time)
    return x, gate, initial, resets, channels // gates if gates else 1


def recurrence(x, gate, initial, resets, *sizes):
    x, gate, state, resets, width = _axes(x, gate, initial, resets, *sizes)
    h = np.empty_like(x)
    with np.errstate(all="ignore"):
        for t in range(x.shape[1]):
            keep, take = _gates(gate[:, t], width)
            h[:, t] = state = keep * np.where(resets[:, t, None], 0, state) + take * x[:, t]
    return h.reshape(-1)


def recurrence_grad(grad, x, gate, h, initial, resets, *sizes):
    x, gate, first, resets, width = _axes(x, gate, initial, resets, *sizes)
    grad, h = _view(grad).reshape(x.shape), _view(h).reshape(x.shape)
    dx, d_gate, after = np.empty_like(x), np.empty_like(gate), np.zeros_like(first)
    with np.errstate(all="ignore"):
        for t in reversed(range(x.shape[1])):
            keep, take = _gates(gate[:, t], width)
            before = np.where(resets[:, t, None], 0, h[:, t - 1] if t else first)
            slope = grad[:, t] + after
            dx[:, t] = slope * take
            each = slope * (before - x[:, t]) * (keep * take)
            d_gate[:, t] = each.reshape(d_gate[:, t].shape + (width,)).sum(-1)
            after = np.where(resets[:, t, None], 0, keep * slope)
    return dx.reshape(-1), d_gate.reshape(-1), None if initial is None else after.reshape(-1)


# ---- causal convolution ----------------------------------------------------------


class _Sequence:
    """Rows of steps with resets and ends."""

    def __init__(self, resets, lengths, batch, time):
        self.resets = np.zeros((batch, time), bool) if resets is None else _view(resets).reshape(batch, time)
        self.ends = np.full(batch, time) if lengths is None else np.clip(_view(lengths).reshape(batch), 0, time)
        self.inside = np.arange(time) < self.ends[:, None]

    def kept(self, array, *axes):
        """An array over (batch, time, ...) with zeros behind the rows' ends."""
        array = _view(array).reshape(self.inside.shape + axes)
        return np.where(self.inside.reshape(self.inside.shape + (1,) * len(axes)), array, 0).astype(array.dtype)


class _Conv(_Sequence):
    def __init__(self, x, weight, bias, initial, resets, lengths, batch, time, channels, taps, activation):
        super().__init__(resets, lengths, batch, time)
        self.x, self.weight, self.taps, self.activation = self.kept(x, channels), _view(weight), taps, activation
        before = np.zeros((batch, taps - 1, channels), self.x.dtype) if initial is None else _view(initial).reshape(batch, taps - 1, channels)
        self.whole = np.concatenate([before, self.x], 1)
        # The step from which on a step sees inputs.
        self.first = np.maximum.accumulate(np.where(self.resets, np.arange(time), -taps), 1)
        with np.errstate(all="ignore"):
            self.pre = np.zeros_like(self.x) if bias is None else np.broadcast_to(_view(bias), self.x.shape)
            for k in range(taps):
                self.pre = self.pre + self.weight[:, k] * self.seen(k)

    def sees(self, k):
        time = self.first.shape[1]
        return (np.arange(time) - (self.taps - 1) + k >= self.first)[..., None]

    def seen(self, k):
        return np.where(self.sees(k), self.whole[:, k : k + self.first.shape[1]], 0)


def causal_conv(x, weight, bias, initial, resets, lengths, *sizes):
    conv = _Conv(x, weight, bias, initial, resets, lengths, *sizes)
    with np.errstate(all="ignore"):
        y = conv.pre * _gates(conv.pre, 1)[0] if conv.activation else conv.pre
    y = np.where(conv.inside[..., None], y, 0).astype(conv.x.dtype)
    last = np.zeros((y.shape[0], conv.taps - 1, y.shape[2]), y.dtype)
    for row, end in enumerate(conv.ends):
        began = conv.first[row, end - 1] if end else -conv.taps
        for k in range(conv.taps - 1):
            if end - (conv.taps - 1) + k >= began:
                last[row, k] = conv.whole[row, end + k]
    return y.reshape(-1), last.reshape(-1)


def causal_conv_grad(grad, x, weight, bias, initial, resets, lengths, *sizes):
    conv = _Conv(x, weight, bias, initial, resets, lengths, *sizes)
    time = conv.first.shape[1]
    d = conv.kept(grad, sizes[2])
    with np.errstate(all="ignore"):
        if conv.activation:
            keep, rest = _gates(conv.pre, 1)
            d = d * (keep * (1 + conv.pre * rest))
            d = np.where(conv.inside[..., None], d, 0).astype(conv.x.dtype)
        d_whole, d_weight = np.zeros_like(conv.whole), np.zeros_like(conv.weight)
        for k in range(conv.taps):
            d_whole[:, k : k + time] += np.where(conv.sees(k), d * conv.weight[:, k], 0)
            d_weight[:, k] = (d * conv.seen(k)).sum((0, 1))
    split = conv.taps - 1
    return [v.reshape(-1) for v in (d_whole[:, split:].copy(), d_weight, d.sum((0, 1)), d_whole[:, :split].copy())]


# ---- selective scan ----------------------------------------------------------------


class _Scan(_Sequence):
    def __init__(self, x, delta, a_log, b, c, skip, gate, initial, delta_bias, resets, lengths, batch, time, channels, groups, states):
        super().__init__(resets, lengths, batch, time)
        self.sizes = batch, time, channels, groups, states
        self.x, delta, self.b, self.c = self.kept(x, channels), self.kept(delta, channels), self.kept(b, groups, states), self.kept(c, groups, states)
        self.skip = None if skip is None else _view(skip)
        self.gate = None if gate is None else self.kept(gate, channels)
        zero = np.zeros((batch, channels, states), self.x.dtype)
        self.initial = zero if initial is None else _view(initial).reshape(zero.shape)
        with np.errstate(all="ignore"):
            self.raw = delta if delta_bias is None else delta + _view(delta_bias)
            self.dt = (np.maximum(self.raw, 0) + np.log1p(np.exp(-np.abs(self.raw)))).astype(self.x.dtype)
            # Past the type's largest number a decay of 0 times an infinite rate would be NaN.
            self.rates = np.minimum(np.exp(_view(a_log)), np.finfo(self.x.dtype).max)

    def wide(self, projected):
        """(batch, groups, states) for every channel."""
        channels, groups = self.sizes[2:4]
        return np.repeat(projected, channels // groups if groups else 1, axis=1)

    def narrow(self, values):
        batch, _, channels, groups, states = self.sizes
        return values.reshape(batch, groups, channels // groups if groups else 1, states).sum(2)

    def step(self, t, state):
        """(states before step t, its decays, states after it)"""
        before = np.where(self.resets[:, t, None, None], 0, state).astype(state.dtype)
        decay = np.exp(-self.dt[:, t, :, None] * self.rates)
        return before, decay, decay * before + (self.dt[:, t] * self.x[:, t])[..., None] * self.wide(self.b[:, t])

    def plain(self, t, after):
        y = (after * self.wide(self.c[:, t])).sum(-1)
        return y if self.skip is None else y + self.skip * self.x[:, t]

    def on(self, t, one, other):
        inside = self.inside[:, t].reshape((-1,) + (1,) * (one.ndim - 1))
        return np.where(inside, one, other).astype(one.dtype)


def selective_scan(*given):
    scan = _Scan(*given)
    state, y = scan.initial, np.zeros_like(scan.x)
    with np.errstate(all="ignore"):
        for t in range(scan.sizes[1]):
            after = scan.step(t, state)[2]
            y[:, t] = scan.on(t, scan.plain(t, after), 0)
            state = scan.on(t, after, state)
        if scan.gate is not None:
            y = np.where(scan.inside[..., None], y * (scan.gate * _gates(scan.gate, 1)[0]), 0).astype(y.dtype)
    return y.reshape(-1), state.reshape(-1).copy()


def selective_scan_grad(grad, grad_state, *given):
    scan = _Scan(*given)
    batch, time, channels, groups, states = scan.sizes
    g = scan.kept(grad, channels)
    state, starts = scan.initial, []
    lam = np.zeros_like(state) if grad_state is None else _view(grad_state).reshape(state.shape)
    dx, d_dt, d_gate = (np.zeros_like(scan.x) for _ in range(3))
    d_b, d_c, d_rates = np.zeros_like(scan.b), np.zeros_like(scan.c), np.zeros_like(scan.rates)
    with np.errstate(all="ignore"):
        for t in range(time):
            before, _, after = scan.step(t, state)
            starts.append(before)
            d_gate[:, t] = scan.on(t, scan.plain(t, after), 0)
            state = scan.on(t, after, state)
        if scan.gate is not None:
            keep, rest = _gates(scan.gate, 1)
            d_gate = np.where(scan.inside[..., None], g * d_gate * (keep * (1 + scan.gate * rest)), 0).astype(g.dtype)
            g = np.where(scan.inside[..., None], g * (scan.gate * keep), 0).astype(g.dtype)
        for t in reversed(range(time)):
            before, decay, after = scan.step(t, starts[t])
            b, c, dt, x, gt = scan.wide(scan.b[:, t]), scan.wide(scan.c[:, t]), scan.dt[:, t], scan.x[:, t], g[:, t]
            here = lam + gt[..., None] * c
            along, share = (here * b).sum(-1), here * (decay * before)
            d_c[:, t] = scan.on(t, scan.narrow(gt[..., None] * after), 0)
            d_b[:, t] = scan.on(t, scan.narrow((dt * x)[..., None] * here), 0)
            dx[:, t] = scan.on(t, along * dt + (0 if scan.skip is None else scan.skip * gt), 0)
            d_dt[:, t] = scan.on(t, along * x - (share * scan.rates).sum(-1), 0)
            d_rates -= scan.on(t, share * dt[..., None], 0).sum(0)
            lam = scan.on(t, np.where(scan.resets[:, t, None, None], 0, decay * here).astype(lam.dtype), lam)
        d_delta = np.where(scan.inside[..., None], d_dt * _gates(scan.raw, 1)[0], 0).astype(d_dt.dtype)
        found = (dx, d_delta, d_rates * scan.rates, d_b, d_c, (g * scan.x).sum((0, 1)), d_gate, d_delta.sum((0, 1)), lam)
    return [v.reshape(-1) for v in found]


# ---- residual stream and norms -------------------------------------------------------


def _inverse_rms(v, eps):
    return 1 / np.sqrt(np.square(v).mean(-1, keepdims=True, dtype=v.dtype) + v.dtype.type(eps))


def _rows(array, rows, channels):
    return _view(array).reshape(rows, channels)


def _factors(gate, scale, rows, channels, divide, dtype):
    if gate is None:
        return dtype.type(scale)
    return np.repeat(_view(gate).reshape(-1, channels), divide, axis=0)[:rows] * dtype.type(scale)


def residual_norm(x, residual, weight, post_weight, gate, rows, channels, divide, scale, eps):
    x, residual = _rows(x, rows, channels), _rows(residual, rows, channels)
    with np.errstate(all="ignore"):
        y = x if post_weight is None else x * _inverse_rms(x, eps) * _view(post_weight)
        stream = residual + _factors(gate, scale, rows, channels, divide, x.dtype) * y
        normed = stream * _inverse_rms(stream, eps) * _view(weight)
    return stream.reshape(-1), normed.reshape(-1)


def residual_norm_grad(grad_stream, grad_normed, x, stream, weight, post_weight, gate, rows, channels, divide, scale, eps):
    ds, dn, x, stream = (_rows(v, rows, channels) for v in (grad_stream, grad_normed, x, stream))
    factor = _factors(gate, scale, rows, channels, divide, x.dtype)
    with np.errstate(all="ignore"):
        outer = _inverse_rms(stream, eps)
        unit, through = stream * outer, dn * _view(weight)
        d_weight = (dn * unit).sum(0)
        d = ds + outer * (through - unit * (through * unit).mean(-1, keepdims=True))
        dx, d_post, y = d * factor, None, x
        if post_weight is not None:
            inner = _inverse_rms(x, eps)
            unit = x * inner
            d_post, through = (dx * unit).sum(0), dx * _view(post_weight)
            y = unit * _view(post_weight)
            dx = inner * (through - unit * (through * unit).mean(-1, keepdims=True))
        d_gate = None
        if gate is not None:
            each = d * y * x.dtype.type(scale)
            d_gate = each.reshape(-1, divide, channels).sum(1) if rows else np.zeros(gate.size, x.dtype)
    return [None if v is None else v.reshape(-1) for v in (dx, d, d_weight, d_post, d_gate)]

# ---- losses from logits ----------------------------------------------------------


class _Rows:
    """Log-probabilities of targets in rows of logits, and the gradient of a weighted sum of them."""

    def __init__(self, logits, targets, mask):
        logits, targets = _view(logits), _view(targets).astype(np.int64)
        self.kept = np.ones(targets.shape, bool) if mask is None else _view(mask)
        self.logits = np.where(self.kept[..., None], logits, 0)
        inside = (targets >= 0) & (targets < logits.shape[-1])
        self.at = np.where(inside, targets, 0)[..., None]
        with np.errstate(all="ignore"):
            top = self.logits.max(-1, keepdims=True)
            self.exp = np.exp(self.logits - top)
            self.total = self.exp.sum(-1, keepdims=True)
            found = (np.take_along_axis(self.logits, self.at, -1) - top - np.log(self.total))[..., 0]
        self.log_probs = np.where(self.kept, np.where(inside, found, np.nan), 0).astype(logits.dtype)

    def grad(self, weights):
        weights = np.where(self.kept, weights, 0).astype(self.logits.dtype)[..., None]
        with np.errstate(all="ignore"):
            grad = self.exp / self.total * -weights
        np.put_along_axis(grad, self.at, np.take_along_axis(grad, self.at, -1) + weights, -1)
        return np.where(self.kept[..., None], grad, 0).astype(self.logits.dtype).reshape(-1)


def token_log_probs(logits, targets, mask):
    return _Rows(logits, targets, mask).log_probs.reshape(-1)


def _grow(x):
    """exp(x) - 1 and exp(x) - 1 - x in 64 bits. Near 0, where a difference would lose the digits of the second, its series."""
    near = np.where(np.abs(x) < 1, x, 0)
    rest = np.ones_like(near)
    for k in range(18, 2, -1):  # x^2/2 (1 + x/3 (1 + x/4 (...)))
        rest = 1 + near / k * rest
    grown = np.expm1(x)
    # Infinite where the policy gives a token no probability; grown - x would be NaN.
    apart = np.where(grown == np.inf, grown, grown - x)
    return grown, np.where(np.abs(x) < 1, near * near / 2 * rest, apart)


def policy_loss(logits, actions, old, advantages, reference, mask, low, high, kl_weight, count, gradient):
    rows = _Rows(logits, actions, mask)
    log_probs, advantages = rows.log_probs, _view(advantages)
    with np.errstate(all="ignore"):
        ratio = np.exp(log_probs - _view(old))
        free = ratio * advantages
        held = np.minimum(np.maximum(ratio, 1 - low), 1 + high) * advantages
        losses, slopes = -np.minimum(free, held), np.where(free > held, 0, -free)
        if reference is not None:
            grown, excess = _grow(_view(reference).astype(np.float64) - log_probs)
            losses, slopes = losses + kl_weight * excess, slopes - kl_weight * grown
        if count is None:
            count = max(1, int(rows.kept.sum()))
        loss = np.asarray(np.where(rows.kept, losses, 0).sum(dtype=np.float64) / count, log_probs.dtype)
        return loss.reshape(-1), log_probs.reshape(-1), rows.grad(slopes / count) if gradient else None


def preference_loss(logits, targets, reference, mask, beta, smoothing, gradient):
    rows = _Rows(logits, targets, mask)
    sums = rows.log_probs.sum(-1)
    pairs = max(1, sums.shape[1])
    with np.errstate(all="ignore"):
        ratios = sums - _view(reference)
        margin = beta * (ratios[0] - ratios[1])
        soft = np.log1p(np.exp(-np.abs(margin)))
        # A side of weight 0 is left out: where a response has probability 0 it is infinite.
        sides = [(1 - smoothing, -margin), (smoothing, margin)]
        losses = sum(weight * (np.maximum(side, 0) + soft) for weight, side in sides if weight)
        yes, no = _gates(margin, 1)
        slope = beta * (smoothing * yes - (1 - smoothing) * no) / pairs
        loss = np.asarray(losses.sum(dtype=np.float64) / pairs, sums.dtype)
        weights = np.stack([slope, -slope])[..., None] * np.ones(rows.kept.shape)
        return loss.reshape(-1), sums.reshape(-1), rows.grad(weights) if gradient else None


def distillation_loss(logits, indices, teacher_logits, teacher_rest, mask, temperature, count, gradient):
    logits, indices, teacher = _view(logits), _view(indices).astype(np.int64), _view(teacher_logits)
    kept = np.ones(indices.shape[:-1], bool) if mask is None else _view(mask)
    dtype, vocab = logits.dtype, logits.shape[-1]
    with np.errstate(all="ignore"):
        # The terms of a list in 64 bits; rows that are left out as zeros. Distances from the list's largest logit
        # are divided by the temperature, as the quotients' own distances would have lost digits.
        t = np.where(kept[..., None], teacher, 0).astype(np.float64)
        base = t.max(-1, keepdims=True)
        base = np.where(base == -np.inf, 0, base)
        t = (t - base) / temperature
        if teacher_rest is not None:
            rest = np.where(kept, _view(teacher_rest), 0).astype(np.longdouble)[..., None]
            t = np.concatenate([t, (rest - base.astype(np.longdouble) / temperature).astype(np.float64)], -1)
        log_p = t - t.max(-1, keepdims=True)
        log_p = log_p - np.log(np.exp(log_p).sum(-1, keepdims=True))
        p = np.exp(log_p)
        logits = np.where(kept[..., None], logits, 0)
        top = logits.max(-1, keepdims=True)
        live = t[..., : indices.shape[-1]] != -np.inf
        named = live & (indices >= 0) & (indices < vocab)
        at = np.where(named, indices, 0)
        apart = (np.take_along_axis(logits, at, -1).astype(np.float64) - top) / temperature
        z = np.exp((logits - top) * dtype.type(1 / temperature))
        total = z.sum(-1, keepdims=True)
        log_total = np.log(total.astype(np.float64))
        log_q = apart - log_total
        listed = np.zeros(z.shape, bool)
        for k in range(indices.shape[-1]):
            one = listed.reshape(-1, vocab)
            one[np.arange(len(one)), at[..., k].reshape(-1)] |= named[..., k].reshape(-1)
        if teacher_rest is not None:
            # Relative to its own largest logit: relative to the row's all of it may be less than the type has.
            others = np.where(listed, -np.inf, logits).astype(dtype)
            other_top = others.max(-1, keepdims=True)
            others = np.exp((others - np.where(other_top == -np.inf, 0, other_top).astype(dtype)) * dtype.type(1 / temperature))
            unlisted = others.sum(-1, keepdims=True)
            log_unlisted = (other_top.astype(np.float64) - top) / temperature + np.log(unlisted.astype(np.float64))
            log_q = np.concatenate([log_q, log_unlisted - log_total], -1)
        losses = np.where(p != 0, p * (log_p - log_q), 0).sum(-1)
        losses = np.where((live & ~named).any(-1) | np.isnan(p).any(-1), np.nan, losses)
        losses = np.where(kept, losses, 0)
        if count is None:
            count = max(1, int(kept.sum()))
        loss = np.asarray(losses.sum() / count, dtype)
        if not gradient:
            return loss.reshape(-1), losses.astype(dtype).reshape(-1), None
        weight = (kept / (count * temperature))[..., None]
        lost = np.isnan(losses)[..., None]
        grad = z / total
        if teacher_rest is not None:
            rest = p[..., -1:]
            grad = grad - np.where(listed | (rest == 0) | (unlisted == 0), 0, rest * (others / unlisted))
        grad = grad * weight
        for k in range(indices.shape[-1]):
            rows = grad.reshape(-1, vocab)
            rows[np.arange(len(rows)), at[..., k].reshape(-1)] -= np.where(named[..., k] & (p[..., k] != 0), p[..., k] * weight[..., 0], 0).reshape(-1)
        grad = np.where(lost, np.nan, grad)
    return loss.reshape(-1), losses.astype(dtype).reshape(-1), np.where(kept[..., None], grad, 0).astype(dtype).reshape(-1)

# ---- AdamW ---------------------------------------------------------------------


def _codes(values, codes, low, positive):
    """Codes of values >= 0 by their share of the block's largest, and that largest: (blocks, BLOCK), (blocks, 1)."""
    blocks = np.pad(values.reshape(-1), (0, -values.size % BLOCK)).reshape(-1, BLOCK)
    with np.errstate(all="ignore"):
        top = blocks.max(1, keepdims=True)
        top = np.where(np.isfinite(top), top, np.float32(np.nan))
        share = blocks / np.where(top > 0, top, np.float32(1))
        # Exact: a power of two scales, and rint rounds ties to even.
        octave = np.where(share > 0, np.maximum(np.frexp(share)[1] - 1, 4 - low), 4 - low)
        steps = np.rint(np.ldexp(share, 4 - octave))
        code = np.where(top > 0, steps + 16 * (octave + low - 4), 0)
        if positive:
            code = np.where(blocks > 0, np.maximum(code, 1), code)
    return np.where(np.isnan(top), 0, code).astype(np.uint8), top


def _share(code, low):
    code = code.astype(np.int32)
    normal = np.ldexp((16 + (code & 15)).astype(np.float32), (code >> 4) - 1 - low)
    return np.where(code < 16, np.ldexp(code.astype(np.float32), -low), normal)


class _Held:
    """Both moments of one tensor in 8 bits."""

    def __init__(self, first, second):
        codes, self.first_top = _codes(np.abs(first), *FIRST, False)
        negative = np.pad(np.signbit(first).reshape(-1), (0, -first.size % BLOCK)).reshape(-1, BLOCK)
        self.first = codes | np.where(negative, 128, 0).astype(np.uint8)
        with np.errstate(all="ignore"):
            self.second, self.second_top = _codes(np.sqrt(second), *SECOND, True)

    def moments(self, shape):
        size = int(np.prod(shape, dtype=np.int64))
        with np.errstate(all="ignore"):
            first = _share(self.first & 127, FIRST[1]) * self.first_top
            first = np.where(self.first & 128, -first, first)
            second = np.square(_share(self.second, SECOND[1]) * self.second_top)
        return [m.reshape(-1)[:size].reshape(shape) for m in (first, second)]


def adamw_load(first, second, shapes, dtype, bits):
    state = []
    for i, shape in enumerate(shapes):
        m, v = (np.zeros(shape, dtype) if given is None else _view(given[i]).copy() for given in (first, second))
        state.append(_Held(m, v) if bits else (m, v))
    return state


def adamw_moments(state, which, shapes, dtype, bits):
    return [(s.moments(shape) if bits else s)[which].reshape(-1).copy() for s, shape in zip(state, shapes)]


def adamw_step(params, grads, state, shapes, dtype, bits, decays, scalars):
    beta1, beta2, step, root, eps = (dtype.type(s) for s in scalars)
    rest1, rest2 = dtype.type(1 - scalars[0]), dtype.type(1 - scalars[1])
    new, after = [], []
    with np.errstate(all="ignore"):
        for p, g, held, shape, decay in zip(params, grads, state, shapes, decays):
            p, g = _view(p), _view(g)
            m, v = held.moments(shape) if bits else held
            m, v = m * beta1 + g * rest1, v * beta2 + g * g * rest2
            new.append((p - (dtype.type(decay) * p + step * m / (np.sqrt(v) * root + eps))).reshape(-1))
            after.append(_Held(m, v) if bits else (m, v))
    return new, after
