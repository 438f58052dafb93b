"""The example that runs the operators of ``nn`` together: it learns its task, on
either backend and with either state, and both backends take the same steps."""

import importlib.util
from pathlib import Path

import numpy as np
import pytest

import openpacho as p

PATH = Path(__file__).resolve().parents[1] / "open-pacho_amd" / "examples" / "recurrent_policy.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("recurrent_policy", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def learns(example, backend, bits):
    episodes = example.Episodes()
    params = example.initial_params(episodes, 32, backend)
    state = p.nn.adamw_state(params, state_bits=bits)
    params, state, rewards = example.train(episodes, params, state, 40)
    # Guesses are right once in five; a learned cue is right almost always.
    assert np.mean(rewards[:3]) < 0.6 and np.mean(rewards[-5:]) > 0.9
    params, state, losses = example.prefer(episodes, params, state, 10)
    assert state.steps == 90 and losses[-1] < np.log(2)
    x, _, _, cues = episodes.draw()
    assert (example.answer(params, x[:, : episodes.length]) == cues[:, 0]).mean() > 0.9


@pytest.mark.parametrize("bits", [None, 8])
def test_it_learns_on_the_host(example, numpy_backend, bits):
    learns(example, numpy_backend, bits)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [None, 8])
def test_it_learns_on_the_device(example, hip, bits):
    learns(example, hip, bits)


@pytest.mark.gpu
def test_both_backends_take_the_same_step(example, hip, numpy_backend):
    found = []
    for backend in (numpy_backend, hip):
        episodes = example.Episodes(seed=3)
        params = example.initial_params(episodes, 16, numpy_backend)
        params = [p.to_backend(a, backend) for a in params]
        x, starts, ends, cues = episodes.draw()
        xs, first, mask = (p.asarray(v, backend=backend) for v in (x, starts, ends))
        values, gates, h, logits = example.forward(params, xs, first)
        old = p.nn.token_log_probs(logits, cues, mask=mask)
        loss, _, d_logits = p.nn.policy_loss_grad(logits, cues, old, np.float32(1.0), mask=mask)
        grads = example.backward(params, xs, first, values, gates, h, d_logits)
        new, state = p.nn.adamw(params, grads, p.nn.adamw_state(params), learning_rate=1e-3)
        found.append([p.asnumpy(a) for a in (loss, d_logits, *grads, *state.first, *new)])
    for one, two in zip(*found):
        # Products of at most 48 x 16 rows in float32 in other orders.
        np.testing.assert_allclose(one, two, rtol=2e-4, atol=2e-5 * max(1e-3, np.abs(one).max()))


def test_the_command(example, capsys):
    assert example.main(["--backend", "numpy", "--steps", "4", "--channels", "8", "--state-bits", "8"]) == 0
    assert "right answers" in capsys.readouterr().out
