"""Operators of ``nn`` on the largest arrays, of nearly 2^31 elements, whose bytes
and whose moments pass 32 bits: the end of one has the bits that it has alone."""

import numpy as np
import pytest

import openpacho as p

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _release(hip):
    yield
    hip.release_cached_memory()


def same(one, two):
    assert one.shape == two.shape
    np.testing.assert_array_equal(p.asnumpy(one), p.asnumpy(two))


def test_recurrence(hip):
    rows, time, channels, heads = 2, 524287, 2048, 8  # of 32 groups of channels a row: one grouping of tiles for both calls
    rng = p.random.default_rng(1, backend=hip)
    x, d = (rng.normal(0, 1, (rows, time, channels), dtype=np.float32) for _ in range(2))
    gate, initial = rng.normal(3, 1, (rows, time, heads), dtype=np.float32), rng.normal(0, 1, (rows, channels), dtype=np.float32)
    h = p.nn.gated_recurrence(x, gate, initial)
    dx, d_gate, d_initial = p.nn.gated_recurrence_grad(d, x, gate, h, initial)
    end = slice(time - 1000, time)
    kept = [a[1:2, end] for a in (h, dx, d_gate)] + [d_initial[1:2]]
    del dx
    last = [a[1:2] for a in (x, gate, initial, d)]
    del x, d, h
    alone = p.nn.gated_recurrence(*last[:3])
    grads = p.nn.gated_recurrence_grad(last[3], last[0], last[1], alone, last[2])
    for got, want in zip(kept, [a[:, end] for a in (alone, *grads[:2])] + [grads[2]]):
        same(got, want)
    # The definition over the last steps, from the state before them.
    state = p.asnumpy(alone[:, end.start - 1]).astype(np.float64)
    xs, a = p.asnumpy(last[0][:, end]).astype(np.float64), 1 / (1 + np.exp(-p.asnumpy(last[1][:, end]).astype(np.float64)))
    a = np.repeat(a, channels // heads, axis=2)
    for t in range(1000):
        state = a[:, t] * state + (1 - a[:, t]) * xs[:, t]
    # 1000 steps of three roundings each, whose weights shrink: some 2^-24 x 10.
    np.testing.assert_allclose(p.asnumpy(kept[0][:, -1]), state, rtol=0, atol=2e-6)


def test_losses(hip):
    rows, vocab, some = 65531, 32769, 200
    rng = p.random.default_rng(2, backend=hip)
    logits = rng.normal(0, 1, (rows, vocab), dtype=np.float32)
    host = np.random.default_rng(2)
    targets, advantages = host.integers(0, vocab, rows), host.standard_normal(rows).astype(np.float32)
    old = np.full(rows, -11, np.float32)
    end = slice(rows - some, rows)
    last = logits[end]
    _, log_probs, grad = p.nn.policy_loss_grad(logits, targets, old, advantages, clip=(1.0, np.inf), count=1.0)
    kept, kept_grad = log_probs[end], grad[end]
    del grad
    _, want, want_grad = p.nn.policy_loss_grad(last, targets[end], old[end], advantages[end], clip=(1.0, np.inf), count=1.0)
    same(kept, want)
    same(kept_grad, want_grad)
    same(p.nn.token_log_probs(logits, targets), log_probs)
    wide = p.asnumpy(last).astype(np.float64)
    exact = wide[np.arange(some), targets[end]] - np.log(np.exp(wide).sum(1))
    np.testing.assert_allclose(p.asnumpy(want), exact, rtol=2e-6)


def test_one_row_of_more_logits(hip):
    vocab = 2**31 - 5
    logits = p.zeros((1, vocab), dtype=np.float32, backend=hip)
    for target in (0, 2**30 + 70, vocab - 1):
        found = p.nn.token_log_probs(logits, [target]).item()
        assert abs(found + np.log(vocab)) < 1e-5  # 2^31 ones add up in a tree: 31 roundings of a float at most
    assert np.isnan(p.nn.token_log_probs(logits, [vocab]).item())


@pytest.mark.parametrize("bits", [None, 8])
def test_adamw(hip, bits):
    size, some = 2**30 + 4396, 4396
    rng = p.random.default_rng(3, backend=hip)
    param, grad = rng.normal(0, 1, (size,), dtype=np.float32), rng.normal(0, 1, (size,), dtype=np.float32)
    end = slice(size - some, size)  # from the start of a block of the quantised moments
    last = param[end], grad[end]
    given = [param[: size - 100], param], [grad[: size - 100], grad]
    options = {"learning_rate": 0.1, "weight_decay": 0.1}
    new, state = p.nn.adamw(*given, p.nn.adamw_state(given[0], state_bits=bits), **options)
    (want,), want_state = p.nn.adamw([last[0]], [last[1]], p.nn.adamw_state([last[0]], state_bits=bits), **options)
    same(new[1][end], want)
    del param, grad, new, given
    for got, alone in ((state.first, want_state.first), (state.second, want_state.second)):
        same(got[1][end], alone[0])
