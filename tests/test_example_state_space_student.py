"""The example that runs the convolution, the selective scan, the residual norm and the distillation loss
together: its gradients against differences, its two backends against each other, its tokens against its rows."""

import importlib.util
from pathlib import Path

import numpy as np
import pytest

import openpacho as p

PATH = Path(__file__).resolve().parents[1] / "open-pacho_amd" / "examples" / "state_space_student.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("state_space_student", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def moved(example, params, direction, by):
    return example.Params(*(p.asarray(p.asnumpy(a) + by * d, backend=a._backend) for a, d in zip(params, direction)))


def gradients_are_slopes(example, backend):
    teacher, params = (example.initial_params(c, n, backend, seed=c, dtype=np.float64) for c, n in ((12, 5), (10, 3)))
    rng = np.random.default_rng(4)
    batch = example.draw(rng, backend, rows=3, steps=9, dtype=np.float64)
    answers = example.teach(teacher, batch)
    _, grads = example.loss_and_grads(params, batch, answers)
    for index, grad in enumerate(grads):
        # One parameter at a time, so that each gradient is seen by itself.
        direction = [np.zeros(a.shape) for a in params]
        direction[index] = rng.standard_normal(grad.shape)
        slope = np.sum(p.asnumpy(grad) * direction[index])
        found = []
        for h in (2e-4, 1e-4):
            up, down = (example.loss_and_grads(moved(example, params, direction, s * h), batch, answers)[0].item() for s in (1, -1))
            found.append((up - down) / (2 * h))
        # Without the differences' error of h^2, which the two tell: 4/3 and -1/3. What is left is of h^4 times a
        # fifth derivative, and rounding: losses near 1 are off by some 1e-14, over h.
        difference = found[1] + (found[1] - found[0]) / 3
        assert abs(slope - difference) <= 1e-8 * (1 + np.sqrt(np.sum(np.square(direction[index])))), params._fields[index]


def test_gradients_are_slopes_on_the_host(example, numpy_backend):
    gradients_are_slopes(example, numpy_backend)


@pytest.mark.gpu
def test_gradients_are_slopes_on_the_device(example, hip):
    gradients_are_slopes(example, hip)


def tokens_are_rows(example, backend):
    params = example.initial_params(20, 6, backend, seed=2, dtype=np.float64)
    x = np.random.default_rng(3).standard_normal((5, 17, example.FEATURES))
    none = np.zeros(x.shape[:2], bool)
    batch = example.Batch(*(p.asarray(v, backend=backend) for v in (x, none, np.full(5, 17), ~none)))
    whole = p.asnumpy(example.forward(params, batch)[0])
    # In double precision other orders of sums of at most 20 products, over 17 steps that forget.
    np.testing.assert_allclose(example.answer(params, x), whole, rtol=0, atol=1e-12 * np.abs(whole).max())


def test_tokens_are_rows_on_the_host(example, numpy_backend):
    tokens_are_rows(example, numpy_backend)


@pytest.mark.gpu
def test_tokens_are_rows_on_the_device(example, hip):
    tokens_are_rows(example, hip)


@pytest.mark.gpu
def test_both_backends_find_the_same(example, hip, numpy_backend):
    found = []
    for backend in (numpy_backend, hip):
        teacher, params = (example.initial_params(c, n, backend, seed=c, dtype=np.float64) for c, n in ((64, 16), (32, 8)))
        batch = example.draw(np.random.default_rng(5), backend, dtype=np.float64)
        if backend is numpy_backend:
            answers = example.teach(teacher, batch)
        loss, grads = example.loss_and_grads(params, batch, answers)
        found.append([p.asnumpy(a) for a in (loss, *grads)])
    for one, two in zip(*found):
        # Double precision; sums of at most 8 x 24 steps in other orders.
        np.testing.assert_allclose(one, two, rtol=0, atol=1e-11 * max(np.abs(one).max(), 1e-3))


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_it_steps_on_the_host(example, numpy_backend, dtype):
    steps(example, numpy_backend, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_it_steps_on_the_device(example, hip, dtype):
    steps(example, hip, dtype)


def steps(example, backend, dtype):
    teacher, params = (example.initial_params(c, n, backend, seed=c, dtype=dtype) for c, n in ((24, 16), (16, 4)))
    batch = example.draw(np.random.default_rng(1), backend, dtype=dtype)
    loss, grads = example.loss_and_grads(params, batch, example.teach(teacher, batch))
    new, state = p.nn.adamw(list(params), list(grads), p.nn.adamw_state(list(params)), learning_rate=1e-2)
    assert loss.dtype == dtype and np.isfinite(loss.item()) and loss.item() > 0 and state.steps == 1
    for before, after in zip(params, new):
        before, after = p.asnumpy(before), p.asnumpy(after)
        assert after.dtype == dtype and np.all(np.isfinite(after)) and np.any(before != after)


def test_the_command(example, capsys):
    assert example.main(["--backend", "numpy", "--steps", "3", "--channels", "8", "--states", "3"]) == 0
    assert "same answers" in capsys.readouterr().out
