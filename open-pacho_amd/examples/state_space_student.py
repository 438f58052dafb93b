"""Distil a state space model into a smaller one, with the operators of ``openpacho.nn``.

Teacher and student are a block on a residual stream between two dense layers:

    stream = x @ w_in
    inner, gate, delta = stream @ w_inner, stream @ w_gate, stream @ w_delta
    u, inputs = causal_conv(inner, w_conv, b_conv, activation="silu")
    y, states = selective_scan(u, delta, a_log, u @ w_b, u @ w_c, skip, gate, delta_bias=bias)
    stream, normed = residual_norm(y @ w_out, stream, w_norm)
    logits = normed @ w_logits

The student sees the teacher's largest logits of each token and the weight of all others
(``distillation_loss``), steps with ``adamw``, and answers one token at a time on the
inputs and states that the steps before left. Rows hold two documents each, separated by a
reset, and end after different numbers of steps.

    python open-pacho_amd/examples/state_space_student.py --backend hip --steps 50
"""

import argparse
import sys
from pathlib import Path
from typing import NamedTuple

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import openpacho as p  # noqa: E402

FEATURES, VOCABULARY, TAPS = 6, 40, 4
nn = p.nn


class Params(NamedTuple):
    w_in: object
    w_inner: object
    w_gate: object
    w_delta: object
    delta_bias: object
    w_conv: object
    b_conv: object
    w_b: object
    w_c: object
    a_log: object
    skip: object
    w_out: object
    w_norm: object
    w_logits: object


def initial_params(channels, states, backend, seed=0, dtype=np.float32):
    """States forget at rates of 1 to ``states`` times their steps, which start near 0.05."""
    rng = np.random.default_rng(seed)

    def matrix(rows, cols):
        return rng.standard_normal((rows, cols)) * rows**-0.5

    square = [matrix(channels, channels) for _ in range(4)]
    values = Params(
        matrix(FEATURES, channels), square[0], square[1], square[2] * 0.1, np.full(channels, -3.0), matrix(TAPS, channels).T,
        np.zeros(channels), matrix(channels, states), matrix(channels, states), np.log(np.tile(np.arange(1.0, states + 1), (channels, 1))),
        np.ones(channels), square[3], np.ones(channels), matrix(channels, VOCABULARY),
    )  # fmt: skip
    return Params(*(p.asarray(np.ascontiguousarray(v.astype(dtype)), backend=backend) for v in values))


class Batch(NamedTuple):
    x: object
    resets: object
    lengths: object
    mask: object  # the steps before each row's end


def draw(rng, backend, rows=8, steps=24, dtype=np.float32):
    lengths = rng.integers(1, steps + 1, rows)
    resets = np.zeros((rows, steps), bool)
    resets[np.arange(rows), rng.integers(0, steps, rows)] = True
    given = rng.standard_normal((rows, steps, FEATURES)).astype(dtype), resets, lengths, np.arange(steps) < lengths[:, None]
    return Batch(*(p.asarray(v, backend=backend) for v in given))


def forward(params, batch):
    """(logits, what ``backward`` needs)."""
    stream = batch.x @ params.w_in
    inner, gate, delta = stream @ params.w_inner, stream @ params.w_gate, stream @ params.w_delta
    u, _ = nn.causal_conv(inner, params.w_conv, params.b_conv, activation="silu", resets=batch.resets, lengths=batch.lengths)
    b, c = (u @ w for w in (params.w_b, params.w_c))
    b, c = (v.reshape(*v.shape[:-1], 1, v.shape[-1]) for v in (b, c))
    given = (u, delta, params.a_log, b, c, params.skip, gate)
    y, _ = nn.selective_scan(*given, delta_bias=params.delta_bias, resets=batch.resets, lengths=batch.lengths)
    out = y @ params.w_out
    after, normed = nn.residual_norm(out, stream, params.w_norm)
    return normed @ params.w_logits, (stream, inner, given, y, out, after, normed)


def _dense_grads(x, weight, grad):
    """Gradients of a layer's input and weight from that of its output."""
    flat_x, flat = x.reshape(-1, x.shape[-1]), grad.reshape(-1, grad.shape[-1])
    return grad @ weight.T, flat_x.T @ flat


def backward(params, batch, kept, d_logits):
    """The parameters' gradients."""
    stream, inner, given, y, out, after, normed = kept
    u = given[0]
    d_normed, d_w_logits = _dense_grads(normed, params.w_logits, d_logits)
    nothing = p.zeros(after.shape, dtype=after.dtype, backend=after._backend)
    d_out, d_stream, d_norm, _, _ = nn.residual_norm_grad(nothing, d_normed, out, after, params.w_norm)
    d_y, d_w_out = _dense_grads(y, params.w_out, d_out)
    d = nn.selective_scan_grad(d_y, *given, delta_bias=params.delta_bias, resets=batch.resets, lengths=batch.lengths)
    d_b, d_c = (v.reshape(*u.shape[:-1], v.shape[-1]) for v in (d.b, d.c))
    through_b, d_w_b = _dense_grads(u, params.w_b, d_b)
    through_c, d_w_c = _dense_grads(u, params.w_c, d_c)
    d_inner, d_conv, d_conv_bias, _ = nn.causal_conv_grad(
        d.x + through_b + through_c, inner, params.w_conv, params.b_conv, activation="silu", resets=batch.resets, lengths=batch.lengths
    )
    d_weights = []
    for weight, grad in ((params.w_inner, d_inner), (params.w_gate, d.gate), (params.w_delta, d.delta)):
        through, d_weight = _dense_grads(stream, weight, grad)
        d_stream = d_stream + through
        d_weights.append(d_weight)
    d_w_in = _dense_grads(batch.x, params.w_in, d_stream)[1]
    return Params(d_w_in, *d_weights, d.delta_bias, d_conv, d_conv_bias, d_w_b, d_w_c, d.a_log, d.skip, d_w_out, d_norm, d_w_logits)


def teach(teacher, batch, entries=8, temperature=2.0):
    """The teacher's answers as it would send them: (indices, logits, log-sum-exp of the rest), on the host."""
    logits = p.asnumpy(forward(teacher, batch)[0])
    indices = np.argsort(-logits, axis=-1, kind="stable")[..., :entries]
    rest = logits / temperature
    np.put_along_axis(rest, indices, -np.inf, axis=-1)
    top = rest.max(-1, keepdims=True)
    rest = np.log(np.exp(rest - top).sum(-1)) + top[..., 0]
    return indices, np.take_along_axis(logits, indices, axis=-1), rest.astype(logits.dtype)


def loss_and_grads(params, batch, answers, temperature=2.0):
    logits, kept = forward(params, batch)
    loss, _, d_logits = nn.distillation_loss_grad(logits, *answers, mask=batch.mask, temperature=temperature)
    return loss, backward(params, batch, kept, d_logits)


def train(teacher, params, state, steps, learning_rate=1e-2, seed=1, log=None):
    """(params, state, losses)."""
    rng, backend, losses = np.random.default_rng(seed), params.w_in._backend, []
    for step in range(steps):
        batch = draw(rng, backend)
        loss, grads = loss_and_grads(params, batch, teach(teacher, batch))
        new, state = nn.adamw(list(params), list(grads), state, learning_rate=learning_rate)
        params = Params(*new)
        losses.append(loss.item())
        if log and step % 20 == 0:
            log(f"step {step}: loss {losses[-1]:.4f}")
    return params, state, losses


def answer(params, x):
    """The logits (rows, steps, vocabulary) of single documents, one token at a time as a server has them."""
    backend, dtype = params.w_in._backend, params.w_in.dtype
    rows, (channels, states) = len(x), params.a_log.shape
    inputs = p.zeros((rows, TAPS - 1, channels), dtype=dtype, backend=backend)
    h = p.zeros((rows, channels, states), dtype=dtype, backend=backend)
    found = []
    for t in range(x.shape[1]):
        stream = p.asarray(np.ascontiguousarray(x[:, t]), backend=backend) @ params.w_in
        u, inputs = nn.causal_conv_step(stream @ params.w_inner, params.w_conv, inputs, params.b_conv, activation="silu")
        b, c = ((u @ w).reshape(rows, 1, states) for w in (params.w_b, params.w_c))
        y, h = nn.selective_scan_step(
            u, stream @ params.w_delta, params.a_log, b, c, h, params.skip, stream @ params.w_gate, delta_bias=params.delta_bias
        )
        _, normed = nn.residual_norm(y @ params.w_out, stream, params.w_norm)
        found.append(p.asnumpy(normed @ params.w_logits))
    return np.stack(found, axis=1)


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--backend", choices=("numpy", "hip"), default="hip")
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--channels", type=int, default=32)
    parser.add_argument("--states", type=int, default=8)
    args = parser.parse_args(argv)
    backend = p.get_backend(args.backend)
    teacher, params = initial_params(2 * args.channels, 16, backend), initial_params(args.channels, args.states, backend, seed=7)
    params, _, losses = train(teacher, params, nn.adamw_state(list(params)), args.steps, log=print)
    x = np.random.default_rng(9).standard_normal((4, 12, FEATURES)).astype(np.float32)
    agree = (answer(params, x).argmax(-1) == answer(teacher, x).argmax(-1)).mean()
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}, same answers {agree:.3f}")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
