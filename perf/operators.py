"""Operators of ``openpacho.nn`` as a training program calls them, for timing and for comparing results.

Four operators: the gated recurrence (with its gradient and its single-token form), the clipped policy loss
and the preference loss from logits (with their gradients), and the AdamW step over many tensors. ``listed()``
names cases over their real range, ``draw(rng)`` gives further ones.

With ``own`` false ``run`` computes them out of elementary torch operations; with ``own`` true it calls
openpacho. Arrays cross between the two as views of one device buffer: torch makes the inputs and reads the
results. Import torch first: the library then shares torch's HIP runtime, so that one device synchronisation
covers both.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

F32, F64 = "float32", "float64"


# ---- the cases -------------------------------------------------------------------


def listed():
    return [
        # One decoding step of 16 sequences: a single token on a carried state. All latency.
        _recurrence("recurrence_step_16x1x2048", F32, 16, 1, 2048, 0, False, False),
        # A training batch of ordinary length with a gate per channel and episode starts inside the rows.
        _recurrence("recurrence_8x4096x2048", F32, 8, 4096, 2048, 0, True, False),
        # Its backward pass: the largest case of the recurrence.
        _recurrence("recurrence_grad_8x4096x2048", F32, 8, 4096, 2048, 0, True, True),
        # One long sequence of odd length, eight heads of 125 channels that share a gate, backward.
        _recurrence("recurrence_grad_1x65537x1000h8", F32, 1, 65537, 1000, 8, False, True),
        # Many tokens over few actions, as a control policy has them: rows of 18 logits.
        _policy("policy_grad_64x257x18", F32, 64, 257, 18, True, False, True),
        # A batch of responses over a vocabulary, with padding and the KL term: the largest logits.
        _policy("policy_grad_16x512x32000", F32, 16, 512, 32000, True, True, True),
        # Few tokens over a large odd vocabulary: rows that have to be split to fill the chip.
        _policy("policy_grad_1x61x151001", F32, 1, 61, 151001, False, True, True),
        # Paired responses of ragged lengths, forward and backward.
        _preference("preference_grad_8x512x32000", F32, 8, 512, 32000, True),
        # A validation batch in double precision, forward only.
        _preference("preference_f64_64x33x1001", F64, 64, 33, 1001, False),
        # A small network of ragged layers: twenty tensors of a few thousand elements, where launches count.
        _adamw("adamw_10x129x65", F32, 0, 10, 129, 65),
        # A large network with full states.
        _adamw("adamw_6x8192x4096", F32, 0, 6, 8192, 4096),
        # The same size class with states in 8 bits and odd extents.
        _adamw("adamw_8bit_8x4097x3001", F32, 8, 8, 4097, 3001),
    ]


def _recurrence(name, dtype, batch, time, channels, heads, resets, grad):
    """heads: 0 for a gate per channel, else the gates that groups of channels share."""
    return {"name": name, "kind": "recurrence", "dtype": dtype, "batch": batch, "time": time, "channels": channels,
            "heads": heads, "resets": resets, "grad": grad}


def _policy(name, dtype, batch, time, vocab, mask, reference, grad):
    return {"name": name, "kind": "policy", "dtype": dtype, "batch": batch, "time": time, "vocab": vocab,
            "mask": mask, "reference": reference, "grad": grad}


def _preference(name, dtype, pairs, time, vocab, grad):
    return {"name": name, "kind": "preference", "dtype": dtype, "pairs": pairs, "time": time, "vocab": vocab,
            "grad": grad}


def _adamw(name, dtype, bits, layers, rows, cols):
    """Per layer a matrix (rows, cols) and a vector (cols,). bits: 8, or 0 for states in the parameters' type."""
    return {"name": name, "kind": "adamw", "dtype": dtype, "bits": bits, "layers": layers, "rows": rows, "cols": cols}


def _size(rng, low, high):
    """A size spread over its logarithm; every other one or so is rounded to a multiple of 16."""
    value = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and value >= 32:
        value = value // 16 * 16
    return max(low, min(high, value))


def _extents(rng, ranges, most):
    """Sizes from (low, high) ranges whose product is at most `most`, none favoured: drawn again until it is."""
    while True:
        sizes = [_size(rng, low, high) for low, high in ranges]
        if math.prod(sizes) <= most:
            return sizes


def draw(rng):
    kind = rng.choice(["recurrence", "recurrence", "policy", "preference", "adamw"])
    dtype = rng.choice([F32, F32, F64])
    half = 2 if dtype == F64 else 1
    grad = rng.random() < 0.6
    if kind == "recurrence":
        heads = _size(rng, 1, 32) if rng.random() < 0.4 else 0
        ranges = [(1, 64), (1, 65537), (1, 4096 // heads if heads else 4096)]
        batch, time, channels = _extents(rng, ranges, (1 << 26) // (half * max(1, heads)))
        case = _recurrence("", dtype, batch, time, channels * max(1, heads), heads, rng.random() < 0.5, grad)
    elif kind == "policy":
        sizes = _extents(rng, [(1, 128), (1, 1024), (2, 160000)], 262144000 // half)
        case = _policy("", dtype, *sizes, rng.random() < 0.7, rng.random() < 0.5, grad)
    elif kind == "preference":
        case = _preference("", dtype, *_extents(rng, [(1, 64), (1, 1024), (2, 64000)], 131072000 // half), grad)
    else:
        layers, rows, cols = _extents(rng, [(1, 10), (1, 8192), (1, 8192)], 6 * 8192 * 4096 // half)
        case = _adamw("", dtype, 0 if dtype == F64 else rng.choice([0, 8]), layers, rows, cols)
    del case["name"]
    return case


# ---- between torch and openpacho ---------------------------------------------------


def _openpacho():
    torch.cuda.is_available()  # torch's HIP runtime is in place before the library loads
    package = str(Path(__file__).resolve().parents[1] / "open-pacho_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import openpacho

    return openpacho


class _View:
    """The device buffer of an openpacho array, as torch takes one in; it keeps the array."""

    def __init__(self, array):
        self.array = array
        self.__cuda_array_interface__ = {
            "shape": array.shape,
            "typestr": array.dtype.str,
            "data": (array._data.ptr, False),
            "version": 2,
        }


def _tensor(array):
    return torch.as_tensor(_View(array), device="cuda")


class _Results(tuple):
    """openpacho's arrays, which whoever reads them gets as torch tensors."""

    def __iter__(self):
        return (_tensor(array) for array in super().__iter__())


def _array(tensor):
    """An openpacho array holding a copy of `tensor`."""
    p = _openpacho()
    hip = p.get_backend("hip")
    array = p.empty(tuple(tensor.shape), dtype=str(tensor.dtype).replace("torch.", ""), backend=hip)
    hip.synchronize()  # the block may come from work that is still queued
    if tensor.numel():
        _tensor(array).copy_(tensor)
    torch.cuda.synchronize()
    return array


# ---- inputs ------------------------------------------------------------------------

_CLIP_LOW, _CLIP_HIGH, _KL_WEIGHT = 0.2, 0.28, 0.04
_BETA, _SMOOTHING = 0.1, 0.05
_RATE, _DECAY, _BETA1, _BETA2, _EPS, _STEPS = 3e-4, 0.1, 0.9, 0.95, 1e-8, 100


def _shapes(case):
    return [(case["rows"], case["cols"]), (case["cols"],)] * case["layers"]


def _inputs(case, seed):
    """The case's inputs as torch tensors, made from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda", dtype=dtype)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    kind = case["kind"]
    if kind == "recurrence":
        # Channels or heads that forget over some steps to some hundreds of steps.
        batch, time, channels, heads = (case[k] for k in ("batch", "time", "channels", "heads"))
        gates = heads or channels
        given = {
            "x": normal(batch, time, channels),
            "gate": normal(batch, time, gates).add_(uniform(gates).mul_(6)),
            "initial": normal(batch, channels),
            "resets": uniform(batch, time) < 1 / 256 if case["resets"] else None,
        }
        if case["grad"]:
            given["h"] = _recurrent(given["x"], given["gate"], given["initial"], given["resets"])
            given["grad"] = normal(batch, time, channels)
        return given
    if kind in ("policy", "preference"):
        lead = (case["batch"], case["time"]) if kind == "policy" else (2, case["pairs"], case["time"])
        logits = normal(*lead, case["vocab"]).mul_(2)
        # Samples of the logits' own distribution, by the largest of logit + Gumbel noise.
        noise = uniform(*lead, case["vocab"]).clamp_(1e-7, 1 - 1e-7).log_().neg_().log_()
        targets = (logits - noise).argmax(-1)
        del noise
        chosen = _log_probs(logits, targets)
        length = torch.ceil(uniform(*lead[:-1], 1) * case["time"])
        steps = torch.arange(case["time"], device="cuda")
        if kind == "policy":
            # Responses end before the rows do; the places after their end hold the action -1.
            mask = (steps < length).expand(lead).contiguous() if case["mask"] else None
            return {
                "logits": logits,
                "actions": targets if mask is None else torch.where(mask, targets, -1),
                "old_log_probs": chosen + 0.2 * normal(*lead),
                "advantages": normal(lead[0], 1),
                "reference_log_probs": chosen + 0.3 * normal(*lead) if case["reference"] else None,
                "mask": mask,
            }
        # The prompt, the first quarter of a row, does not count.
        mask = ((steps < length) & (steps >= case["time"] // 4)).contiguous()
        sums = torch.where(mask, chosen, torch.zeros_like(chosen)).sum(-1)
        return {"logits": logits, "targets": targets, "reference_log_probs": sums + 4 * normal(*lead[:-1]), "mask": mask}
    given = {"params": [], "grads": [], "first": [], "second": []}
    for shape in _shapes(case):
        scale = 1e-2 * torch.exp(normal(shape[-1]))  # gradients differ by column
        given["params"].append(normal(*shape).mul_(0.02))
        given["grads"].append(normal(*shape).mul_(scale))
        first, second = normal(*shape).mul_(scale).mul_(0.3), normal(*shape).mul_(scale).square_()
        if case["bits"]:
            first, second = _held([first], _held_first)[0], _held([second], _held_second)[0]
        given["first"].append(first)
        given["second"].append(second)
    return given


def prepare(case, seed):
    given = _inputs(case, seed)
    if own:
        p = _openpacho()
        given = {
            name: [_array(t) for t in value] if isinstance(value, list) else None if value is None else _array(value)
            for name, value in given.items()
        }
        if case["kind"] == "adamw":
            given["state"] = p.nn.adamw_state(
                given["params"], state_bits=case["bits"] or None, steps=_STEPS, first=given.pop("first"),
                second=given.pop("second"),
            )
        torch.cuda.synchronize()
    return {"case": case, "given": given}


# ---- the work ----------------------------------------------------------------------


def run(state):
    case, given = state["case"], state["given"]
    work = {"recurrence": _run_recurrence, "policy": _run_policy, "preference": _run_preference, "adamw": _run_adamw}
    return work[case["kind"]](case, **given)


def _run_recurrence(case, x, gate, initial, resets, h=None, grad=None):
    if own:
        nn = _openpacho().nn
        if case["grad"]:
            return _Results(nn.gated_recurrence_grad(grad, x, gate, h, initial, resets=resets))
        return _Results([nn.gated_recurrence(x, gate, initial, resets=resets)])
    if case["grad"]:
        return _recurrent_grad(grad, x, gate, h, initial, resets)
    return (_recurrent(x, gate, initial, resets),)


def _run_policy(case, logits, actions, old_log_probs, advantages, reference_log_probs, mask):
    if own:
        nn = _openpacho().nn
        loss = nn.policy_loss_grad if case["grad"] else nn.policy_loss
        return _Results(
            loss(logits, actions, old_log_probs, advantages, reference_log_probs=reference_log_probs, mask=mask,
                 clip=(_CLIP_LOW, _CLIP_HIGH), kl_weight=_KL_WEIGHT if case["reference"] else 0.0)
        )
    kept = torch.ones_like(old_log_probs) if mask is None else mask.to(logits.dtype)
    actions = actions.clamp(min=0)
    log_probs, shifted, total = _log_softmax_at(logits, actions)
    ratio = torch.exp(log_probs - old_log_probs)
    plain = ratio * advantages
    clipped = ratio.clamp(1 - _CLIP_LOW, 1 + _CLIP_HIGH) * advantages
    losses = -torch.minimum(plain, clipped)
    slope = -torch.where(plain <= clipped, plain, torch.zeros_like(plain))
    if reference_log_probs is not None:
        difference = reference_log_probs - log_probs
        grown = torch.exp(difference)
        losses = losses + _KL_WEIGHT * (grown - difference - 1)
        slope = slope + _KL_WEIGHT * (1 - grown)
    count = kept.sum().clamp(min=1)
    loss = (losses * kept).sum() / count
    log_probs = log_probs * kept
    if not case["grad"]:
        return loss, log_probs
    return loss, log_probs, _logits_grad(shifted, total, actions, slope * kept / count)


def _run_preference(case, logits, targets, reference_log_probs, mask):
    if own:
        nn = _openpacho().nn
        loss = nn.preference_loss_grad if case["grad"] else nn.preference_loss
        return _Results(loss(logits, targets, reference_log_probs, mask=mask, beta=_BETA, smoothing=_SMOOTHING))
    kept = mask.to(logits.dtype)
    log_probs, shifted, total = _log_softmax_at(logits, targets)
    sums = (log_probs * kept).sum(-1)
    ratios = sums - reference_log_probs
    margin = _BETA * (ratios[0] - ratios[1])
    # -log sigma(x) = max(-x, 0) + log(1 + exp(-|x|))
    soft = torch.log1p(torch.exp(-margin.abs()))
    losses = (1 - _SMOOTHING) * ((-margin).clamp(min=0) + soft) + _SMOOTHING * (margin.clamp(min=0) + soft)
    pairs = margin.shape[0]
    loss = losses.sum() / pairs
    if not case["grad"]:
        return loss, sums
    slope = _BETA / pairs * (_SMOOTHING * torch.sigmoid(margin) - (1 - _SMOOTHING) * torch.sigmoid(-margin))
    weights = torch.stack([slope, -slope])[..., None] * kept
    return loss, sums, _logits_grad(shifted, total, targets, weights)


def _run_adamw(case, params, grads, first=None, second=None, state=None):
    if own:
        new, after = _openpacho().nn.adamw(
            params, grads, state, learning_rate=_RATE, betas=(_BETA1, _BETA2), eps=_EPS, weight_decay=_DECAY
        )
        return {"params": _Results(new), "first": _Results(after.first), "second": _Results(after.second)}
    shapes = [t.shape for t in params]
    sizes = [t.numel() for t in params]
    p, g, m, v = (torch.cat([t.reshape(-1) for t in given]) for given in (params, grads, first, second))
    one, two = 1 - _BETA1 ** (_STEPS + 1), 1 - _BETA2 ** (_STEPS + 1)
    m = m * _BETA1 + g * (1 - _BETA1)
    v = v * _BETA2 + g * g * (1 - _BETA2)
    p = p * (1 - _RATE * _DECAY) - m * (_RATE / one) / (torch.sqrt(v) * (1 / math.sqrt(two)) + _EPS)
    p, m, v = ([t.view(shape) for t, shape in zip(flat.split(sizes), shapes)] for flat in (p, m, v))
    if case["bits"]:
        m, v = _held(m, _held_first), _held(v, _held_second)
    return {"params": p, "first": m, "second": v}


# ---- plain forms of the parts --------------------------------------------------------


def _scanned(a, b):
    """h_t = a_t h_{t-1} + b_t along axis 1 from h = 0, by doubling the reach of every element."""
    reach = 1
    while reach < a.shape[1]:
        b = torch.cat([b[:, :reach], a[:, reach:] * b[:, :-reach] + b[:, reach:]], 1)
        a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], 1)
        reach *= 2
    return b


def _gates(gate, channels):
    """sigma(gate) and 1 - sigma(gate) of every channel."""
    gate = gate.repeat_interleave(channels // gate.shape[-1], dim=-1)
    return torch.sigmoid(gate), torch.sigmoid(-gate)


def _recurrent(x, gate, initial, resets):
    keep, take = _gates(gate, x.shape[-1])
    if resets is not None:
        keep = torch.where(resets[..., None], torch.zeros_like(keep), keep)
    b = take * x
    b[:, :1] += keep[:, :1] * initial[:, None]
    return _scanned(keep, b)


def _recurrent_grad(grad, x, gate, h, initial, resets):
    keep, take = _gates(gate, x.shape[-1])
    before = torch.cat([initial[:, None], h[:, :-1]], 1)
    passed = keep
    if resets is not None:
        passed = torch.where(resets[..., None], torch.zeros_like(keep), keep)
        before = torch.where(resets[..., None], torch.zeros_like(before), before)
    # mu_t = a_t (grad_t + mu_{t+1}), from the last step to the first.
    carried = _scanned(passed.flip(1), (passed * grad).flip(1)).flip(1)
    slope = grad + torch.cat([carried[:, 1:], torch.zeros_like(carried[:, :1])], 1)
    d_gate = slope * (before - x) * (keep * take)
    heads = gate.shape[-1]
    d_gate = d_gate.view(*d_gate.shape[:-1], heads, -1).sum(-1)
    return slope * take, d_gate, carried[:, 0]


def _log_softmax_at(logits, index):
    """log-probabilities at `index`, exp(logits - max) and its sums over the last axis."""
    top = logits.amax(-1, keepdim=True)
    shifted = torch.exp(logits - top)
    total = shifted.sum(-1, keepdim=True)
    at = torch.gather(logits, -1, index[..., None])
    return (at - top - torch.log(total))[..., 0], shifted, total


def _log_probs(logits, index):
    return _log_softmax_at(logits, index)[0]


def _logits_grad(shifted, total, index, weights):
    weights = weights[..., None]
    d_logits = shifted * (-weights / total)
    return d_logits.scatter_add_(-1, index[..., None], weights)


_BLOCK = 256  # elements of a tensor that share a scale


def _held(tensors, rule):
    """The values that 8-bit codes of each tensor stand for: blocks of _BLOCK elements, the last one shorter."""
    blocks = [torch.nn.functional.pad(t.reshape(-1), (0, -t.numel() % _BLOCK)).view(-1, _BLOCK) for t in tensors]
    held = rule(torch.cat(blocks)).split([len(b) for b in blocks])
    return [h.reshape(-1)[: t.numel()].view(t.shape) for h, t in zip(held, tensors)]


def _rounded(y, lowest):
    """y in [0, 1], float32, to the nearest value of four mantissa bits and exponents of `lowest` or more (ties to even)."""
    exponent = ((y.view(torch.int32) >> 23) - 127).clamp(min=lowest)
    quantum = ((exponent - 4 + 127) << 23).view(torch.float32)
    return torch.round(y / quantum) * quantum


def _fractions(values, lowest):
    """values >= 0 over their block's largest, rounded, and that largest."""
    top = values.amax(1, keepdim=True)
    return torch.where(top > 0, _rounded(values / torch.where(top > 0, top, torch.ones_like(top)), lowest), 0.0), top


def _held_first(m):
    fraction, top = _fractions(m.abs(), -6)
    return torch.sign(m) * fraction * top


def _held_second(v):
    root = torch.sqrt(v)
    fraction, top = _fractions(root, -14)
    fraction = torch.where(root > 0, fraction.clamp(min=2.0**-18), fraction)
    return torch.square(fraction * top)


def work(case):
    """Bytes: each input read once and each output written once. Operations: a few for each element."""
    size = np.dtype(case["dtype"]).itemsize
    kind = case["kind"]
    if kind == "recurrence":
        steps = case["batch"] * case["time"]
        count, gates, state = steps * case["channels"], steps * (case["heads"] or case["channels"]), case["batch"] * case["channels"]
        moved = 4 * count + 2 * gates + 2 * state if case["grad"] else 2 * count + gates + state
        return {"bytes": size * moved + (steps if case["resets"] else 0), "flops": (20 if case["grad"] else 12) * count}
    if kind in ("policy", "preference"):
        rows = case["batch"] * case["time"] if kind == "policy" else 2 * case["pairs"] * case["time"]
        count = rows * case["vocab"]
        return {"bytes": size * count * (2 if case["grad"] else 1) + 8 * rows, "flops": (5 if case["grad"] else 3) * count}
    count = case["layers"] * (case["rows"] + 1) * case["cols"]
    if case["bits"]:
        # Parameters, gradients, codes and scales in; parameters, codes and scales out, and the values of the codes.
        return {"bytes": (3 * 4 + 4 + 2 * 4) * count + 4 * 4 * count // _BLOCK, "flops": 30 * count}
    return {"bytes": 7 * size * count, "flops": 14 * count}


# ---- the same in 64 bits -------------------------------------------------------------


def exact(case, seed):
    given = _inputs(case, seed)
    made = {"recurrence": _exact_recurrence, "policy": _exact_policy, "preference": _exact_preference, "adamw": _exact_adamw}
    return made[case["kind"]](case, **given)


def _exact_recurrence(case, x, gate, initial, resets, h=None, grad=None):
    """Step by step, as the definition has it."""
    batch, time, channels = x.shape
    width = channels // gate.shape[-1]
    x, gate, initial = x.double(), gate.double(), initial.double()

    def step(t):
        a = (1 / (1 + torch.exp(-gate[:, t]))).repeat_interleave(width, dim=1)
        b = (1 / (1 + torch.exp(gate[:, t]))).repeat_interleave(width, dim=1)
        goes_on = 1.0 if resets is None else (~resets[:, t : t + 1]).double()
        return a, b, goes_on

    if not case["grad"]:
        out, now = torch.empty_like(x), initial
        for t in range(time):
            a, b, goes_on = step(t)
            now = a * (now * goes_on) + b * x[:, t]
            out[:, t] = now
        return [out]
    h, grad = h.double(), grad.double()
    dx, d_gate, after = torch.empty_like(x), torch.empty_like(gate), torch.zeros_like(initial)
    for t in reversed(range(time)):
        a, b, goes_on = step(t)
        previous = (h[:, t - 1] if t else initial) * goes_on
        slope = grad[:, t] + after
        dx[:, t] = slope * b
        d_gate[:, t] = (slope * (previous - x[:, t]) * a * b).view(batch, -1, width).sum(2)
        after = slope * a * goes_on
    return [dx, d_gate, after]


def _exact_policy(case, logits, actions, old_log_probs, advantages, reference_log_probs, mask):
    rows = torch.ones_like(actions, dtype=torch.bool) if mask is None else mask
    logits = logits.double()
    actions = torch.where(rows, actions, 0)
    log_p = torch.log_softmax(logits, -1)
    del logits
    at = log_p.gather(-1, actions.unsqueeze(-1)).squeeze(-1)
    ratio = (at - old_log_probs.double()).exp()
    gain = advantages.double().expand_as(ratio)
    # With a gain above zero the ratio stops counting over 1 + high, with one below zero under 1 - low.
    stops = torch.where(gain > 0, ratio > 1 + _CLIP_HIGH, (ratio < 1 - _CLIP_LOW) & (gain < 0))
    limit = (gain > 0).double() * (_CLIP_HIGH + _CLIP_LOW) + (1 - _CLIP_LOW)
    each = torch.where(stops, -limit * gain, -ratio * gain)
    slope = torch.where(stops, 0.0, -ratio * gain)
    if reference_log_probs is not None:
        q = reference_log_probs.double() - at
        each = each + _KL_WEIGHT * (torch.expm1(q) - q)
        slope = slope - _KL_WEIGHT * torch.expm1(q)
    count = max(1, int(rows.sum()))
    loss = each[rows].sum() / count
    outputs = [loss, torch.where(rows, at, 0.0)]
    if case["grad"]:
        weights = torch.where(rows, slope / count, 0.0).unsqueeze(-1)
        d_logits = log_p.exp_().mul_(-weights)
        outputs.append(d_logits.scatter_add_(-1, actions.unsqueeze(-1), weights))
    return outputs


def _exact_preference(case, logits, targets, reference_log_probs, mask):
    log_p = torch.log_softmax(logits.double(), -1)
    at = log_p.gather(-1, targets.unsqueeze(-1)).squeeze(-1)
    sums = torch.where(mask, at, 0.0).sum(-1)
    margin = _BETA * ((sums[0] - sums[1]) - (reference_log_probs[0].double() - reference_log_probs[1].double()))
    good, bad = torch.nn.functional.logsigmoid(margin), torch.nn.functional.logsigmoid(-margin)
    outputs = [-((1 - _SMOOTHING) * good + _SMOOTHING * bad).mean(), sums]
    if case["grad"]:
        slope = -_BETA * ((1 - _SMOOTHING) * bad.exp() - _SMOOTHING * good.exp()) / case["pairs"]
        weights = (torch.stack((slope, -slope)).unsqueeze(-1) * mask).unsqueeze(-1)
        d_logits = log_p.exp_().mul_(-weights)
        outputs.append(d_logits.scatter_add_(-1, targets.unsqueeze(-1), weights))
    return outputs


def _exact_adamw(case, params, grads, first, second):
    t = _STEPS + 1
    found = {"params": [], "first": [], "second": []}
    for p, g, m, v in zip(params, grads, first, second):
        p, g, m, v = p.double(), g.double(), m.double(), v.double()
        m = _BETA1 * m + (1 - _BETA1) * g
        v = _BETA2 * v + (1 - _BETA2) * g.square()
        step = (m / (1 - _BETA1**t)) / ((v / (1 - _BETA2**t)).sqrt() + _EPS)
        found["params"].append(p - _RATE * step - _RATE * _DECAY * p)
        if case["bits"]:
            m = m.sign() * _nearest(m.abs(), 112, 10, False)
            v = _nearest(v.sqrt(), 240, 18, True).square()
        found["first"].append(m)
        found["second"].append(v)
    return found


def _nearest(values, codes, low, positive):
    """values in 64 bits, each the nearest of the `codes` fractions of its block's largest value; `positive`: a
    value above zero takes the smallest fraction at least."""
    grid = torch.tensor(
        [c * 2.0**-low if c < 16 else (16 + c % 16) * 2.0 ** (c // 16 - 1 - low) for c in range(codes + 1)],
        dtype=torch.float64, device=values.device,
    )
    flat = torch.nn.functional.pad(values.reshape(-1), (0, -values.numel() % _BLOCK)).view(-1, _BLOCK)
    top = flat.amax(1, keepdim=True)
    share = flat / top.clamp(min=torch.finfo(torch.float64).tiny)
    code = torch.bucketize(share, (grid[1:] + grid[:-1]) / 2)
    if positive:
        code = torch.where(share > 0, code.clamp(min=1), code)
    return (grid[code] * top).reshape(-1)[: values.numel()].view(values.shape)
