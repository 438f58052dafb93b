"""Further operators of ``openpacho.nn`` as a program calls them, for timing and for comparing results.

Four operators of a state space block and of its training: the short causal convolution, the selective scan (each
for sequences, for their gradients and for single tokens), the residual stream with the norms after and before
a block, and the loss against a teacher's top logits. ``listed()`` names cases over their real range, ``draw(rng)``
gives further ones.

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
        # One decoding step of 16 sequences on carried states: all latency.
        _scan("scan_step_16x2048n16", F32, "step", 16, 1, 2048, 16, 1),
        # Prompts of ragged lengths, whose last states go on to single tokens.
        _scan("scan_8x2048x2048n16", F32, "forward", 8, 2048, 2048, 16, 1, lengths=True),
        # A training batch of packed episodes, backward: the largest case of the scan.
        _scan("scan_grad_8x2048x2048n16", F32, "grad", 8, 2048, 2048, 16, 1, resets=True),
        # One long sequence of odd length, four groups of 250 channels with projections of their own.
        _scan("scan_grad_1x16387x1000n16g4", F32, "grad", 1, 16387, 1000, 16, 4),
        # The convolution of one decoding step.
        _conv("conv_step_16x2048w4", F32, "step", 16, 1, 2048, 4),
        # A long sequence of odd channels through a convolution of three steps, ragged inside a batch of two.
        _conv("conv_2x16387x1001w3", F32, "forward", 2, 16387, 1001, 3, lengths=True),
        # A training batch, backward.
        _conv("conv_grad_8x4096x2048w4", F32, "grad", 8, 4096, 2048, 4, resets=True),
        # The residual stream of one decoding step.
        _norm("norm_16x1x2048", F32, False, 16, 1, 2048, "channel"),
        # A training batch with a gate for each token and channel, backward: the largest of its kind.
        _norm("norm_grad_8x4096x2048", F32, True, 8, 4096, 2048, "token"),
        # Odd rows, a gate for each sequence, in double precision.
        _norm("norm_grad_f64_3x1367x1537", F64, True, 3, 1367, 1537, "sequence"),
        # A batch of responses over a vocabulary with the teacher's 64 largest logits and the rest of its mass.
        _distill("distill_grad_16x512x32000k64", F32, True, 16, 512, 32000, 64, True),
        # Few tokens over a large odd vocabulary, the teacher's list alone.
        _distill("distill_grad_1x61x151001k20", F32, True, 1, 61, 151001, 20, False),
    ]


def _scan(name, dtype, kind, batch, time, channels, states, groups, resets=False, lengths=False):
    return {"name": name, "op": "scan", "dtype": dtype, "kind": kind, "batch": batch, "time": time, "channels": channels,
            "states": states, "groups": groups, "resets": resets, "lengths": lengths}


def _conv(name, dtype, kind, batch, time, channels, taps, resets=False, lengths=False):
    return {"name": name, "op": "conv", "dtype": dtype, "kind": kind, "batch": batch, "time": time, "channels": channels,
            "taps": taps, "resets": resets, "lengths": lengths}


def _norm(name, dtype, grad, batch, time, channels, gate):
    """gate: none, or one factor per "channel", per "sequence" and channel, per "token" and channel."""
    return {"name": name, "op": "norm", "dtype": dtype, "grad": grad, "batch": batch, "time": time, "channels": channels, "gate": gate}


def _distill(name, dtype, grad, batch, time, vocab, top, rest):
    return {"name": name, "op": "distill", "dtype": dtype, "grad": grad, "batch": batch, "time": time, "vocab": vocab, "top": top,
            "rest": rest}


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
    op = rng.choice(["scan", "scan", "conv", "norm", "distill"])
    dtype = rng.choice([F32, F32, F64])
    half = 2 if dtype == F64 else 1
    if op in ("scan", "conv"):
        kind = rng.choice(["forward", "grad", "grad", "step"])
        resets, lengths = rng.random() < 0.4, rng.random() < 0.4
        if kind == "step":
            resets = lengths = False
    if op == "scan":
        states, groups = rng.choice([1, 4, 8, 16, 16, 32, 64]), rng.choice([1, 1, 2, 4])
        ranges = [(1, 64), (1, 1 if kind == "step" else 16387), (1, 4096 // groups)]
        # Fewer in double precision, where an exponential is a small program.
        batch, time, channels = _extents(rng, ranges, (1 << 28) // (4 if dtype == F64 else 1) // (states * groups))
        case = _scan("", dtype, kind, batch, time, channels * groups, states, groups, resets, lengths)
    elif op == "conv":
        batch, time, channels = _extents(rng, [(1, 64), (1, 1 if kind == "step" else 65537), (1, 4096)], (1 << 26) // half)
        case = _conv("", dtype, kind, batch, time, channels, rng.randint(2, 5), resets, lengths)
    elif op == "norm":
        sizes = _extents(rng, [(1, 64), (1, 8192), (1, 16384)], (1 << 26) // half)
        case = _norm("", dtype, rng.random() < 0.6, *sizes, rng.choice(["none", "channel", "sequence", "token"]))
    else:
        batch, time, vocab = _extents(rng, [(1, 64), (1, 1024), (8, 160000)], 262144000 // half)
        case = _distill("", dtype, rng.random() < 0.6, batch, time, vocab, min(vocab, _size(rng, 1, 128)), rng.random() < 0.5)
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

_SCALE, _EPS = 0.5, 1e-6
_TEMPERATURE = 2.0


def _inputs(case, seed):
    """The case's inputs as torch tensors, made from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda", dtype=dtype)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    op, batch, time = case["op"], case["batch"], case["time"]
    if op in ("scan", "conv"):
        channels, kind = case["channels"], case["kind"]
        lead = (batch,) if kind == "step" else (batch, time)
        sequences = {
            # Episodes of some hundreds of steps, packed; prompts that end before the batch's longest does.
            "resets": uniform(batch, time) < 1 / 256 if case["resets"] else None,
            "lengths": torch.ceil(uniform(batch) * time).to(torch.int64) if case["lengths"] else None,
        }
    if op == "scan":
        states, groups = case["states"], case["groups"]
        # Steps from a thousandth to a tenth, moved by the input; states that forget at rates 1, 2, 3, ...
        step = torch.exp(uniform(channels) * math.log(100.0) + math.log(1e-3))
        given = {
            "x": normal(*lead, channels),
            "delta": normal(*lead, channels).mul_(0.5),
            "a_log": torch.log(torch.arange(1, states + 1, device="cuda", dtype=dtype)).repeat(channels, 1) + 0.1 * normal(channels, states),
            "b": normal(*lead, groups, states),
            "c": normal(*lead, groups, states),
            "skip": 1 + 0.1 * normal(channels),
            "gate": normal(*lead, channels),
            "initial": normal(batch, channels, states).mul_(0.5),
            "delta_bias": step + torch.log(-torch.expm1(-step)),
            **sequences,
        }
        if kind == "grad":
            given["grad"] = normal(*lead, channels)
        return given
    if op == "conv":
        taps = case["taps"]
        given = {
            "x": normal(*lead, channels),
            "weight": normal(channels, taps).mul_(taps**-0.5),
            "bias": normal(channels).mul_(0.1),
            "initial": normal(batch, taps - 1, channels),
            **sequences,
        }
        if kind == "grad":
            given["grad"] = normal(*lead, channels)
        return given
    if op == "norm":
        channels = case["channels"]
        shape = {"none": None, "channel": (channels,), "sequence": (batch, 1, channels), "token": (batch, time, channels)}[case["gate"]]
        given = {
            "x": normal(batch, time, channels).mul_(0.7),
            "residual": normal(batch, time, channels).mul_(2),
            "weight": 1 + 0.1 * normal(channels),
            "post_weight": 1 + 0.1 * normal(channels),
            "gate": None if shape is None else 0.5 + 0.3 * normal(*shape),
        }
        if case["grad"]:
            # A step backward has the stream of the step forward in place of the residual.
            given["stream"] = _residual_norm(given["x"], given.pop("residual"), given["weight"], given["post_weight"], given["gate"])[0]
            given["grad_stream"], given["grad_normed"] = normal(batch, time, channels), normal(batch, time, channels)
        return given
    vocab, top = case["vocab"], case["top"]
    logits = normal(batch, time, vocab).mul_(2)
    # A teacher that agrees with the student in part.
    teacher = normal(batch, time, vocab).mul_(2).add_(logits)
    teacher_logits, indices = torch.topk(teacher, top, dim=-1)
    # What its other logits add up to.
    rest = torch.logsumexp(teacher.scatter_(-1, indices, -math.inf) / _TEMPERATURE, dim=-1) if case["rest"] else None
    length = torch.ceil(uniform(batch, 1) * time)
    return {
        "logits": logits,
        "indices": indices,
        "teacher_logits": teacher_logits,
        "teacher_rest": rest,
        "mask": (torch.arange(time, device="cuda") < length).contiguous(),
    }


def prepare(case, seed):
    given = _inputs(case, seed)
    if own:
        given = {name: None if value is None else _array(value) for name, value in given.items()}
        torch.cuda.synchronize()
    return {"case": case, "given": given}


# ---- the work ----------------------------------------------------------------------


def run(state):
    case, given = state["case"], state["given"]
    return {"scan": _run_scan, "conv": _run_conv, "norm": _run_norm, "distill": _run_distill}[case["op"]](case, **given)


def _run_scan(case, x, delta, a_log, b, c, skip, gate, initial, delta_bias, resets, lengths, grad=None):
    if own:
        nn = _openpacho().nn
        if case["kind"] == "step":
            return _Results(nn.selective_scan_step(x, delta, a_log, b, c, initial, skip, gate, delta_bias=delta_bias))
        given, options = (x, delta, a_log, b, c, skip, gate, initial), dict(delta_bias=delta_bias, resets=resets, lengths=lengths)
        if case["kind"] == "grad":
            return _Results(nn.selective_scan_grad(grad, *given, **options))
        return _Results(nn.selective_scan(*given, **options))
    if case["kind"] == "step":
        x, delta, b, c, gate = (v[:, None] for v in (x, delta, b, c, gate))
    valid = _valid(x, lengths)
    width = x.shape[-1] // b.shape[2]
    if valid is not None:
        x, gate = (torch.where(valid[..., None], v, torch.zeros_like(v)) for v in (x, gate))
        b, c = (torch.where(valid[..., None, None], v, torch.zeros_like(v)) for v in (b, c))
    b, c = (v.repeat_interleave(width, dim=2) if width != 1 else v for v in (b, c))
    raw = delta + delta_bias
    dt = raw.clamp(min=0) + torch.log1p(torch.exp(-raw.abs()))
    if valid is not None:
        dt = torch.where(valid[..., None], dt, torch.zeros_like(dt))
    a = -torch.exp(a_log)
    decay = torch.exp(dt[..., None] * a)
    if resets is not None:
        cut = resets if valid is None else resets & valid
        decay = torch.where(cut[..., None, None], torch.zeros_like(decay), decay)
    u = (dt * x)[..., None] * b
    u[:, :1] += decay[:, :1] * initial[:, None]
    h = _scanned(decay, u)
    del u
    y = (h * c).sum(-1) + skip * x
    if case["kind"] != "grad":
        y = y * (gate * torch.sigmoid(gate))
        return (y[:, 0] if case["kind"] == "step" else y), h[:, -1].contiguous()
    if valid is not None:
        grad = torch.where(valid[..., None], grad, torch.zeros_like(grad))
    sig = torch.sigmoid(gate)
    d_gate = grad * y * (sig * (1 + gate * (1 - sig)))
    g = grad * (gate * sig)
    # lam_t = c_t g_t + decay_{t+1} lam_{t+1}
    after = torch.cat([decay[:, 1:], torch.zeros_like(decay[:, :1])], 1).flip(1)
    lam = _scanned(after, (c * g[..., None]).flip(1)).flip(1)
    del after
    d_c = _group_sums(g[..., None] * h, width)
    d_b = _group_sums((dt * x)[..., None] * lam, width)
    along = (lam * b).sum(-1)
    d_initial = decay[:, 0] * lam[:, 0]
    before = torch.cat([initial[:, None], h[:, :-1]], 1)
    q = lam * decay * before  # a reset's decay is 0
    del lam, before, h, decay
    d_raw = ((q * a).sum(-1) + along * x) * torch.sigmoid(raw)
    if valid is not None:
        d_raw = torch.where(valid[..., None], d_raw, torch.zeros_like(d_raw))
    d_a_log = (q * dt[..., None]).sum((0, 1)) * a
    return along * dt + skip * g, d_raw, d_a_log, d_b, d_c, (g * x).sum((0, 1)), d_gate, d_raw.sum((0, 1)), d_initial


def _run_conv(case, x, weight, bias, initial, resets, lengths, grad=None):
    if own:
        nn = _openpacho().nn
        if case["kind"] == "step":
            return _Results(nn.causal_conv_step(x, weight, initial, bias, activation="silu"))
        options = dict(resets=resets, lengths=lengths, activation="silu")
        if case["kind"] == "grad":
            return _Results(nn.causal_conv_grad(grad, x, weight, bias, initial, **options))
        return _Results(nn.causal_conv(x, weight, bias, initial, **options))
    if case["kind"] == "step":
        x = x[:, None]
    taps, time = weight.shape[1], x.shape[1]
    whole = torch.cat([initial, x], 1)
    valid = _valid(x, lengths)
    pre = torch.zeros_like(x) + bias
    sees = []
    for back in range(taps):  # the input `back` steps before
        seen = whole[:, taps - 1 - back : taps - 1 - back + time]
        keep = _reaches(resets, back)
        sees.append(seen if keep is None else torch.where(keep[..., None], seen, torch.zeros_like(seen)))
        pre = pre + weight[:, taps - 1 - back] * sees[-1]
    sig = torch.sigmoid(pre)
    if case["kind"] != "grad":
        y = pre * sig
        if valid is not None:
            y = torch.where(valid[..., None], y, torch.zeros_like(y))
        return (y[:, 0] if case["kind"] == "step" else y), _window(whole, taps, resets, lengths)
    d_pre = grad * (sig * (1 + pre * (1 - sig)))
    if valid is not None:
        d_pre = torch.where(valid[..., None], d_pre, torch.zeros_like(d_pre))
    d_whole, d_weight = torch.zeros_like(whole), torch.empty_like(weight)
    for back, seen in enumerate(sees):
        keep = _reaches(resets, back)
        part = d_pre * weight[:, taps - 1 - back]
        d_whole[:, taps - 1 - back : taps - 1 - back + time] += part if keep is None else torch.where(keep[..., None], part, torch.zeros_like(part))
        d_weight[:, taps - 1 - back] = (d_pre * seen).sum((0, 1))
    return d_whole[:, taps - 1 :].contiguous(), d_weight, d_pre.sum((0, 1)), d_whole[:, : taps - 1].contiguous()


def _run_norm(case, x, weight, post_weight, gate, residual=None, stream=None, grad_stream=None, grad_normed=None):
    if own:
        nn, options = _openpacho().nn, dict(post_weight=post_weight, gate=gate, scale=_SCALE, eps=_EPS)
        if case["grad"]:
            found = nn.residual_norm_grad(grad_stream, grad_normed, x, stream, weight, **options)
            return _Results([v for v in found if v is not None])
        return _Results(nn.residual_norm(x, residual, weight, **options))
    if not case["grad"]:
        return _residual_norm(x, residual, weight, post_weight, gate)
    n = x.shape[-1]
    inner = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS)
    outer = 1 / torch.sqrt((stream * stream).mean(-1, keepdim=True) + _EPS)
    unit = stream * outer
    d_weight = (grad_normed * unit).sum((0, 1))
    through = grad_normed * weight
    d = grad_stream + outer * (through - unit * ((through * unit).sum(-1, keepdim=True) / n))
    factor = _SCALE if gate is None else _SCALE * gate
    unit = x * inner
    d_post = d * factor
    d_post_weight = (d_post * unit).sum((0, 1))
    through = d_post * post_weight
    dx = inner * (through - unit * ((through * unit).sum(-1, keepdim=True) / n))
    if gate is None:
        return dx, d, d_weight, d_post_weight
    d_gate = d * (_SCALE * post_weight) * unit
    if gate.dim() == 1:
        d_gate = d_gate.sum((0, 1))
    elif gate.shape[1] != d_gate.shape[1]:
        d_gate = d_gate.sum(1, keepdim=True)
    return dx, d, d_weight, d_post_weight, d_gate


def _run_distill(case, logits, indices, teacher_logits, teacher_rest, mask):
    if own:
        nn = _openpacho().nn
        loss = nn.distillation_loss_grad if case["grad"] else nn.distillation_loss
        return _Results(loss(logits, indices, teacher_logits, teacher_rest, mask=mask, temperature=_TEMPERATURE))
    t = teacher_logits / _TEMPERATURE
    if teacher_rest is not None:  # the rest as one class
        t = torch.cat([t, teacher_rest[..., None]], -1)
    log_p = t - t.amax(-1, keepdim=True)
    log_p = log_p - torch.log(torch.exp(log_p).sum(-1, keepdim=True))
    p = torch.exp(log_p)
    z = logits / _TEMPERATURE
    top = z.amax(-1, keepdim=True)
    at = torch.gather(logits, -1, indices) / _TEMPERATURE - top
    z = torch.exp(z - top)
    total = z.sum(-1, keepdim=True)
    log_q = at - torch.log(total)
    if teacher_rest is not None:
        unlisted = z.scatter(-1, indices, 0.0).sum(-1, keepdim=True)
        log_q = torch.cat([log_q, torch.log(unlisted) - torch.log(total)], -1)
    losses = torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p)).sum(-1)
    losses = torch.where(mask, losses, torch.zeros_like(losses))
    kept = mask.to(z.dtype)
    count = kept.sum().clamp(min=1)
    loss = losses.sum() / count
    if not case["grad"]:
        return loss, losses
    weight = (kept / (count * _TEMPERATURE))[..., None]
    if teacher_rest is None:
        return loss, losses, (z * (weight / total)).scatter_add_(-1, indices, -p * weight)
    p, rest = p[..., :-1], p[..., -1:]
    rest = torch.where(rest > 0, rest / unlisted, torch.zeros_like(rest))
    here = (torch.gather(z, -1, indices) / total - p) * weight
    return loss, losses, (z * ((1 / total - rest) * weight)).scatter_(-1, indices, here)


# ---- plain forms of the parts --------------------------------------------------------


def _scanned(a, b):
    """h_t = a_t h_{t-1} + b_t along axis 1 from h = 0, by doubling the reach of every element."""
    reach = 1
    while reach < a.shape[1]:
        b = torch.cat([b[:, :reach], a[:, reach:] * b[:, :-reach] + b[:, reach:]], 1)
        a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], 1)
        reach *= 2
    return b


def _group_sums(values, width):
    batch, time, channels, states = values.shape
    return values.view(batch, time, channels // width, width, states).sum(3)


def _valid(x, lengths):
    return None if lengths is None else torch.arange(x.shape[1], device=x.device) < lengths[:, None]


def _reaches(resets, back):
    """Whether a step sees the one `back` steps before it: no reset from there on, its own among them."""
    if resets is None or not back:
        return None
    keep = ~resets
    for k in range(1, back):
        keep = keep & ~torch.cat([torch.zeros_like(resets[:, :k]), resets[:, : -k or None][:, : resets.shape[1] - k]], 1)
    return keep


def _window(whole, taps, resets, lengths):
    """The last taps - 1 inputs before each row's end, those before its last reset as zeros."""
    batch, time = whole.shape[0], whole.shape[1] - (taps - 1)
    ends = torch.full((batch,), time, device=whole.device, dtype=torch.int64) if lengths is None else lengths
    at = ends[:, None] + torch.arange(taps - 1, device=whole.device)
    found = torch.gather(whole, 1, at[..., None].expand(-1, -1, whole.shape[2]))
    if resets is not None:
        steps = torch.arange(time, device=whole.device)
        last = torch.where(resets & (steps < ends[:, None]), steps, -taps).amax(1)
        found = torch.where((at - (taps - 1) >= last[:, None])[..., None], found, torch.zeros_like(found))
    return found


def _residual_norm(x, residual, weight, post_weight, gate):
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS) * post_weight
    stream = residual + _SCALE * (y if gate is None else gate * y)
    return stream, stream / torch.sqrt((stream * stream).mean(-1, keepdim=True) + _EPS) * weight


def work(case):
    """Bytes: each input read once and each output written once. Operations: a few for each element."""
    size = np.dtype(case["dtype"]).itemsize
    op, batch, time = case["op"], case["batch"], case["time"]
    tokens = batch * time
    if op == "scan":
        channels, states = case["channels"], case["states"]
        wide, narrow, state = tokens * channels, 2 * tokens * case["groups"] * states, batch * channels * states
        if case["kind"] == "grad":
            return {"bytes": size * (7 * wide + 2 * narrow + 2 * state), "flops": 24 * wide * states}
        return {"bytes": size * (4 * wide + narrow + 2 * state), "flops": 8 * wide * states}
    if op == "conv":
        wide, window = tokens * case["channels"], batch * (case["taps"] - 1) * case["channels"]
        if case["kind"] == "grad":
            return {"bytes": size * (3 * wide + 2 * window), "flops": (6 * case["taps"] + 10) * wide}
        return {"bytes": size * (2 * wide + 2 * window), "flops": (2 * case["taps"] + 6) * wide}
    if op == "norm":
        wide = tokens * case["channels"]
        gated = {"none": 0, "channel": 0, "sequence": 0, "token": 1}[case["gate"]] * wide
        if case["grad"]:
            return {"bytes": size * (6 * wide + 2 * gated), "flops": 24 * wide}
        return {"bytes": size * (4 * wide + gated), "flops": 10 * wide}
    count, top = tokens * case["vocab"], tokens * case["top"]
    return {"bytes": size * count * (2 if case["grad"] else 1) + (size + 8) * top, "flops": (6 if case["grad"] else 4) * count}


# ---- the same in 64 bits -------------------------------------------------------------


def exact(case, seed):
    given = {k: v.double() if v is not None and v.is_floating_point() else v for k, v in _inputs(case, seed).items()}
    return {"scan": _exact_scan, "conv": _exact_conv, "norm": _exact_norm, "distill": _exact_distill}[case["op"]](case, **given)


def _exact_scan(case, x, delta, a_log, b, c, skip, gate, initial, delta_bias, resets, lengths, grad=None):
    """Step by step, as the definition has it."""
    if case["kind"] == "step":
        x, delta, b, c, gate = (v.unsqueeze(1) for v in (x, delta, b, c, gate))
    batch, time, channels = x.shape
    groups = b.shape[2]
    rates = -a_log.exp()
    dt = torch.nn.functional.softplus(delta + delta_bias, threshold=700)
    on = torch.ones((batch, time), dtype=torch.bool, device=x.device) if lengths is None else torch.arange(time, device=x.device) < lengths[:, None]
    cut = torch.zeros_like(on) if resets is None else resets

    def wide(v):  # (batch, groups, states) for every channel
        return v[:, :, None].expand(-1, -1, channels // groups, -1).reshape(batch, channels, -1)

    y, state = torch.zeros_like(x), initial
    past = [] if case["kind"] == "grad" else None
    for t in range(time):
        if past is not None:
            past.append(torch.where(cut[:, t, None, None], 0.0, state))
        start = torch.where(cut[:, t, None, None], 0.0, state)
        after = (dt[:, t, :, None] * rates).exp() * start + (dt[:, t] * x[:, t])[..., None] * wide(b[:, t])
        state = torch.where(on[:, t, None, None], after, state)
        y[:, t] = torch.where(on[:, t, None], (after * wide(c[:, t])).sum(-1) + skip * x[:, t], 0.0)
    silu = gate * gate.sigmoid()
    if case["kind"] != "grad":
        y = y * silu
        return [y[:, 0] if case["kind"] == "step" else y, state]
    dx, d_dt, d_b, d_c = (torch.zeros_like(v) for v in (x, x, b, c))
    d_rates, lam = torch.zeros_like(rates), torch.zeros_like(initial)
    g = torch.where(on[..., None], grad * silu, 0.0)
    for t in reversed(range(time)):
        live = on[:, t, None]
        bt, ct = wide(b[:, t]), wide(c[:, t])
        decay = (dt[:, t, :, None] * rates).exp()
        h = decay * past[t] + (dt[:, t] * x[:, t])[..., None] * bt
        here = lam + g[:, t, :, None] * ct
        d_c[:, t] = torch.where(live[..., None], (g[:, t, :, None] * h).view(batch, groups, -1, h.shape[-1]).sum(2), 0.0)
        d_b[:, t] = torch.where(live[..., None], (here * (dt[:, t] * x[:, t])[..., None]).view(batch, groups, -1, h.shape[-1]).sum(2), 0.0)
        share = here * decay * past[t]
        dx[:, t] = torch.where(live, (here * bt).sum(-1) * dt[:, t] + skip * g[:, t], 0.0)
        d_dt[:, t] = torch.where(live, (share * rates).sum(-1) + (here * bt).sum(-1) * x[:, t], 0.0)
        d_rates += torch.where(live[..., None], share * dt[:, t, :, None], 0.0).sum(0)
        passed = torch.where(cut[:, t, None, None], 0.0, decay * here)
        lam = torch.where(live[..., None], passed, lam)
        past[t] = None
    d_delta = d_dt * (delta + delta_bias).sigmoid()
    d_gate = grad * y * (gate.sigmoid() + silu * (1 - gate.sigmoid()))
    return [dx, d_delta, d_rates * rates, d_b, d_c, (g * x).sum((0, 1)), d_gate, d_delta.sum((0, 1)), lam]


def _exact_conv(case, x, weight, bias, initial, resets, lengths, grad=None):
    """Each step's window of inputs as an axis of its own."""
    if case["kind"] == "step":
        x = x.unsqueeze(1)
    batch, time, channels = x.shape
    taps = weight.shape[1]
    ends = [time] * batch if lengths is None else lengths.tolist()
    padded = torch.cat((initial, x), 1)
    # first[t]: the step from which on step t sees inputs, counted in x; at row's starts it sees the carried ones.
    steps = torch.arange(time, device=x.device)
    first = torch.full((batch, time), -taps, device=x.device)
    if resets is not None:
        first = torch.cummax(torch.where(resets, steps, -taps), 1).values
    windows = padded.unfold(1, taps, 1)  # (batch, time, channels, taps)
    at = steps[:, None] + torch.arange(1 - taps, 1, device=x.device)
    sees = (at >= first[..., None])[:, :, None]
    on = steps < torch.tensor(ends, device=x.device)[:, None]
    y, outputs = torch.empty_like(x), None
    for row in range(batch):  # by rows, for the windows' memory
        pre = (torch.where(sees[row], windows[row], 0.0) * weight).sum(-1) + bias
        y[row] = pre
    s = y.sigmoid()
    if case["kind"] != "grad":
        out = torch.where(on[..., None], y * s, 0.0)
        state = torch.zeros_like(initial)
        for row, end in enumerate(ends):
            state[row] = padded[row, end : end + taps - 1]
            if end and taps > 1:
                began = int(first[row, end - 1])
                for k in range(taps - 1):
                    if end - (taps - 1) + k < began:
                        state[row, k] = 0
        return [out[:, 0] if case["kind"] == "step" else out, state]
    d_pre = torch.where(on[..., None], grad * (s + y * s * (1 - s)), 0.0)
    d_padded, d_weight = torch.zeros_like(padded), torch.zeros_like(weight)
    for row in range(batch):
        d_weight += (torch.where(sees[row], windows[row], 0.0) * d_pre[row, ..., None]).sum(0)
        for k in range(taps):
            d_padded[row, k : k + time] += torch.where(sees[row, :, :, k], d_pre[row] * weight[:, k], 0.0)
    return [d_padded[:, taps - 1 :], d_weight, d_pre.sum((0, 1)), d_padded[:, : taps - 1]]


def _exact_norm(case, x, weight, post_weight, gate, residual=None, stream=None, grad_stream=None, grad_normed=None):
    factor = _SCALE * (torch.ones_like(weight) if gate is None else gate)
    if not case["grad"]:
        out = residual + factor * post_weight * x * (x.square().mean(-1, keepdim=True) + _EPS).rsqrt()
        return [out, out * weight * (out.square().mean(-1, keepdim=True) + _EPS).rsqrt()]
    scale2 = (stream.square().mean(-1, keepdim=True) + _EPS).rsqrt()
    d = grad_stream + scale2 * weight * grad_normed - scale2**3 * stream * (stream * weight * grad_normed).mean(-1, keepdim=True)
    scale1 = (x.square().mean(-1, keepdim=True) + _EPS).rsqrt()
    w = factor * post_weight * d
    dx = scale1 * w - scale1**3 * x * (x * w).mean(-1, keepdim=True)
    found = [dx, d, (grad_normed * stream * scale2).sum((0, 1)), (factor * d * x * scale1).sum((0, 1))]
    if gate is not None:
        each = _SCALE * post_weight * d * x * scale1
        found.append({"channel": lambda: each.sum((0, 1)), "sequence": lambda: each.sum(1, keepdim=True), "token": lambda: each}[case["gate"]]())
    return found


def _exact_distill(case, logits, indices, teacher_logits, teacher_rest, mask):
    log_q = torch.log_softmax(logits / _TEMPERATURE, -1)
    t = teacher_logits / _TEMPERATURE
    whole = torch.logsumexp(t, -1)
    if teacher_rest is not None:
        whole = torch.logaddexp(whole, teacher_rest)
    log_p = t - whole.unsqueeze(-1)
    p = log_p.exp()
    each = (p * (log_p - log_q.gather(-1, indices))).sum(-1)
    q = log_q.exp_()
    if teacher_rest is not None:
        others = q.scatter(-1, indices, 0.0)
        unlisted, log_rest = others.sum(-1), teacher_rest - whole
        rest = log_rest.exp()
        each = each + torch.where(rest > 0, rest * (log_rest - unlisted.log()), 0.0)
        if case["grad"]:
            q -= others * torch.where(rest > 0, rest / unlisted, 0.0).unsqueeze(-1)
        del others
    each = torch.where(mask, each, 0.0)
    count = max(1, int(mask.sum()))
    if not case["grad"]:
        return [each.sum() / count, each]
    grad = q.scatter_add_(-1, indices, -p) * (mask / (count * _TEMPERATURE)).unsqueeze(-1)
    return [each.sum() / count, each, grad]
