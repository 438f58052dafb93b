"""Train a recurrent policy to recall a cue, with the operators of ``openpacho.nn``.

Each sequence shows one of ``symbols`` cues in its first step and noise afterwards;
in the last step the policy answers with a symbol. The policy is a gated recurrence
between two dense layers:

    values, gates = x @ w_v + b_v, x @ w_g + b_g
    h = gated_recurrence(values, gates)
    logits = h @ w_o + b_o

``train`` improves it by the clipped policy loss from its own answers, whose reward
is 1 for the cue; ``prefer`` continues from pairs of a right and a wrong answer, by the
preference loss. Both step with ``adamw``. Rows hold two episodes each, separated by a
reset.

    python open-pacho_amd/examples/recurrent_policy.py --backend hip --state-bits 8
"""

import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import openpacho as p  # noqa: E402


class Episodes:
    """Batches of cue sequences: inputs, where episodes start, where they answer, and the answers."""

    def __init__(self, symbols=5, length=8, batch=48, seed=0):
        self.symbols, self.length, self.batch = symbols, length, batch
        self.features = symbols + 2
        self.rng = np.random.default_rng(seed)

    def draw(self):
        rows, steps = self.batch, 2 * self.length
        x = np.zeros((rows, steps, self.features), np.float32)
        x[..., self.symbols :] = self.rng.standard_normal((rows, steps, 2))
        cues = self.rng.integers(0, self.symbols, (rows, 2))
        starts, ends = np.zeros((rows, steps), bool), np.zeros((rows, steps), bool)
        for episode in range(2):
            first = episode * self.length
            x[np.arange(rows), first, cues[:, episode]] = 3
            starts[:, first], ends[:, first + self.length - 1] = True, True
        return x, starts, ends, np.repeat(cues, self.length, axis=1)


def initial_params(episodes, channels, backend, seed=1):
    """[w_v, b_v, w_g, b_g, w_o, b_o]; the gates start mostly open towards the past."""
    rng = p.random.default_rng(seed, backend=backend)
    features, symbols = episodes.features, episodes.symbols

    def matrix(rows, cols):
        return rng.normal(0, rows**-0.5, (rows, cols), dtype=np.float32)

    def vector(size, value):
        return p.full((size,), value, dtype=np.float32, backend=backend)

    return [matrix(features, channels), vector(channels, 0), matrix(features, channels), vector(channels, 1),
            matrix(channels, symbols), vector(symbols, 0)]  # fmt: skip


def forward(params, x, starts):
    w_v, b_v, w_g, b_g, w_o, b_o = params
    values, gates = x @ w_v + b_v, x @ w_g + b_g
    h = p.nn.gated_recurrence(values, gates, resets=starts)
    return values, gates, h, h @ w_o + b_o


def _dense_grads(x, grad):
    """Gradients of a layer's weights and bias from those of its output, (rows, steps, n)."""
    x, grad = x.reshape(-1, x.shape[-1]), grad.reshape(-1, grad.shape[-1])
    return x.T @ grad, grad.sum(axis=0)


def backward(params, x, starts, values, gates, h, d_logits):
    d_values, d_gates, _ = p.nn.gated_recurrence_grad(d_logits @ params[4].T, values, gates, h, resets=starts)
    return [*_dense_grads(x, d_values), *_dense_grads(x, d_gates), *_dense_grads(h, d_logits)]


def _sample(logits, rng):
    """Answers drawn from the logits' distribution on the host."""
    return (logits - np.log(-np.log(rng.random(logits.shape)))).argmax(-1)


def train(episodes, params, state, steps, learning_rate=3e-2, log=None):
    """Policy steps on answers drawn from the policy itself, two for each batch; (params, state, mean rewards)."""
    backend, rewards = params[0]._backend, []
    for step in range(steps):
        x, starts, ends, cues = episodes.draw()
        x, starts, mask = (p.asarray(v, backend=backend) for v in (x, starts, ends))
        logits = forward(params, x, starts)[-1]
        actions = _sample(p.asnumpy(logits), episodes.rng)
        reward = (actions == cues).astype(np.float32)
        rewards.append(float(reward[ends].mean()))
        advantages = reward - rewards[-1]
        old = p.nn.token_log_probs(logits, actions, mask=mask)
        for _ in range(2):
            values, gates, h, logits = forward(params, x, starts)
            loss, _, d_logits = p.nn.policy_loss_grad(
                logits, actions, old, advantages, reference_log_probs=old, mask=mask, kl_weight=0.01
            )
            grads = backward(params, x, starts, values, gates, h, d_logits)
            params, state = p.nn.adamw(params, grads, state, learning_rate=learning_rate, weight_decay=1e-4)
        if log and step % 20 == 0:
            log(f"policy step {step}: reward {rewards[-1]:.3f}, loss {loss.item():.4f}")
    return params, state, rewards


def prefer(episodes, params, state, steps, learning_rate=1e-2, log=None):
    """Preference steps on pairs of the right and a wrong answer; (params, state, losses)."""
    backend, losses = params[0]._backend, []
    for step in range(steps):
        x, starts, ends, cues = episodes.draw()
        wrong = (cues + episodes.rng.integers(1, episodes.symbols, cues.shape)) % episodes.symbols
        targets, masks = np.stack([cues, wrong]), np.stack([ends, ends])
        x, starts = p.asarray(x, backend=backend), p.asarray(starts, backend=backend)
        values, gates, h, logits = forward(params, x, starts)
        rows, length, symbols = logits.shape
        # Both answers see the same sequence: its logits once for each, and their gradients added.
        both = p.asarray(np.zeros((2, 1, 1, 1), np.float32), backend=backend) + logits
        loss, _, d_both = p.nn.preference_loss_grad(both, targets, np.zeros((2, rows), np.float32), mask=masks, beta=0.5)
        grads = backward(params, x, starts, values, gates, h, d_both.sum(axis=0))
        params, state = p.nn.adamw(params, grads, state, learning_rate=learning_rate, weight_decay=1e-4)
        losses.append(loss.item())
        if log and step % 20 == 0:
            log(f"preference step {step}: loss {losses[-1]:.4f}")
    return params, state, losses


def answer(params, x):
    """The answers to single sequences, one token at a time on a carried state, as a server has them."""
    backend = params[0]._backend
    w_v, b_v, w_g, b_g, w_o, b_o = params
    h = p.zeros((len(x), w_v.shape[1]), dtype=np.float32, backend=backend)
    for t in range(x.shape[1]):
        token = p.asarray(np.ascontiguousarray(x[:, t]), backend=backend)
        h = p.nn.gated_recurrence_step(token @ w_v + b_v, token @ w_g + b_g, h)
    return p.asnumpy(h @ w_o + b_o).argmax(-1)


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--backend", choices=("numpy", "hip"), default="hip")
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--channels", type=int, default=32)
    parser.add_argument("--state-bits", type=int, choices=(8,), default=None)
    args = parser.parse_args(argv)
    episodes = Episodes()
    params = initial_params(episodes, args.channels, p.get_backend(args.backend))
    state = p.nn.adamw_state(params, state_bits=args.state_bits)
    params, state, rewards = train(episodes, params, state, args.steps, log=print)
    params, state, losses = prefer(episodes, params, state, args.steps // 2, log=print)
    x, _, _, cues = episodes.draw()
    right = (answer(params, x[:, : episodes.length]) == cues[:, 0]).mean()
    print(f"reward {np.mean(rewards[-10:]):.3f}, preference loss {np.mean(losses[-10:]):.4f}, right answers {right:.3f}")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
