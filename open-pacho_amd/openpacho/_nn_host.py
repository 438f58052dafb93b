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
