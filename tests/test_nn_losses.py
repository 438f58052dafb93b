"""The losses of ``nn`` on the NumPy backend: values and gradients against the
definitions, gradients against differences, masks, and what they refuse."""

import numpy as np
import pytest

import openpacho as p
from oracle import training


def within(got, want, units, dtype):
    got = p.asnumpy(got)
    assert got.dtype == dtype and got.shape == np.shape(want)
    error = np.abs(got.astype(training.WIDE) - want)
    bound = units * np.finfo(dtype).eps / 2 + np.finfo(dtype).tiny
    assert np.all(error <= bound), float(np.max(error / bound))


def policy_inputs(rows, vocab, dtype, seed=0, masked=True, reference=True, index=np.int64):
    rng = np.random.default_rng(seed)
    logits = (3 * rng.standard_normal((rows, vocab))).astype(dtype)
    mask = rng.random(rows) < 0.7 if masked else None
    actions = rng.integers(0, vocab, rows).astype(index)
    near = np.array([float(training.Row(z, y).log_prob) for z, y in zip(logits, actions)])
    old = (near + 0.3 * rng.standard_normal(rows)).astype(dtype)
    ref = (near + 0.5 * rng.standard_normal(rows)).astype(dtype) if reference else None
    advantages = rng.standard_normal(rows).astype(dtype)
    if masked:
        # What a mask leaves out may hold anything.
        out = np.flatnonzero(~mask)
        actions[out] = rng.choice([-1, vocab, 2**31 - 1, -(2**31)], len(out))
        logits[out[::2]], old[out], advantages[out] = np.nan, np.inf, np.nan
        if ref is not None:
            ref[out] = -np.inf
    return logits, actions, old, advantages, ref, mask


def put(backend, *values):
    return [None if v is None else p.asarray(v, backend=backend) for v in values]


def check_policy(backend, rows, vocab, dtype, seed=0, masked=True, reference=True, index=np.int64, **options):
    given = policy_inputs(rows, vocab, dtype, seed, masked, reference, index)
    logits, actions, old, advantages, ref, mask = put(backend, *given)
    clip = options.get("clip", 0.2)
    ends = clip if isinstance(clip, tuple) else (clip, clip)
    weight = options.setdefault("kl_weight", 0.05 if reference else 0.0)
    values, units, undecided = training.policy_loss(*given[:4], given[4], given[5], ends, weight, options.get("count"))
    found = p.nn.policy_loss_grad(logits, actions, old, advantages, reference_log_probs=ref, mask=mask, **options)
    # Where rounding decides on which side of the clip a ratio is, the gradient may be either side's; the loss is continuous there.
    assert undecided.sum() <= max(1, rows // 500)
    for got, want, unit in zip(found[:2], values, units):
        within(got, want, unit, dtype)
    decided = ~undecided
    within(p.asarray(p.asnumpy(found[2])[decided]), values[2][decided], units[2][decided], dtype)
    if mask is not None:
        out = ~given[5]
        assert not p.asnumpy(found[1])[out].any() and not p.asnumpy(found[2])[out].any()
    for got, same in zip(p.nn.policy_loss(logits, actions, old, advantages, reference_log_probs=ref, mask=mask, **options), found):
        np.testing.assert_array_equal(p.asnumpy(got), p.asnumpy(same))
    alone = p.nn.token_log_probs(logits, actions, mask=mask)
    np.testing.assert_array_equal(p.asnumpy(alone), p.asnumpy(found[1]))


def preference_inputs(pairs, time, vocab, dtype, seed=0, index=np.int64):
    rng = np.random.default_rng(seed)
    logits = (2 * rng.standard_normal((2, pairs, time, vocab))).astype(dtype)
    targets = rng.integers(0, vocab, (2, pairs, time)).astype(index)
    length = rng.integers(0, time + 1, (2, pairs, 1))
    mask = (np.arange(time) < length) & (np.arange(time) > 0)
    targets[~mask] = -100
    logits[~mask] = np.inf
    sums = training.preference_loss(logits, targets, np.zeros((2, pairs)), mask)[0][1].astype(float)
    return logits, targets, (sums + 5 * rng.standard_normal((2, pairs))).astype(dtype), mask


def check_preference(backend, pairs, time, vocab, dtype, seed=0, index=np.int64, **options):
    given = preference_inputs(pairs, time, vocab, dtype, seed, index)
    logits, targets, reference, mask = put(backend, *given)
    values, units = training.preference_loss(*given, **options)
    found = p.nn.preference_loss_grad(logits, targets, reference, mask=mask, **options)
    for got, want, unit in zip(found, values, units):
        within(got, want, unit, dtype)
    for got, same in zip(p.nn.preference_loss(logits, targets, reference, mask=mask, **options), found):
        np.testing.assert_array_equal(p.asnumpy(got), p.asnumpy(same))


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 7), (9, 2), (40, 33), (5, 300)])
def test_policy_loss(numpy_backend, rows, vocab, dtype):
    check_policy(numpy_backend, rows, vocab, dtype, seed=rows)
    check_policy(numpy_backend, rows, vocab, dtype, seed=vocab, masked=False, reference=False, index=np.int32)
    check_policy(numpy_backend, rows, vocab, dtype, clip=(0.1, np.inf), count=7, kl_weight=0.5)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("pairs,time,vocab", [(1, 1, 3), (3, 5, 7), (2, 9, 64)])
def test_preference_loss(numpy_backend, pairs, time, vocab, dtype):
    check_preference(numpy_backend, pairs, time, vocab, dtype, seed=pairs)
    check_preference(numpy_backend, pairs, time, vocab, dtype, beta=0.5, smoothing=0.1, index=np.int32)


def differences(value, logits, step=1e-6):
    found = np.empty_like(logits)
    for at in np.ndindex(logits.shape):
        ends = []
        for sign in (1, -1):
            moved = logits.copy()
            moved[at] += sign * step
            ends.append(value(moved))
        found[at] = (ends[0] - ends[1]) / (2 * step)
    return found


def test_gradients_match_differences(numpy_backend):
    logits, actions, old, advantages, reference, _ = policy_inputs(6, 5, np.float64, 2, masked=False)
    mask = np.array([True, False, True, True, True, False])
    arguments, options = (actions, old, advantages), dict(reference_log_probs=reference, mask=mask, kl_weight=0.3, clip=(0.1, 0.4))
    ends = training.policy_loss(logits, *arguments, reference, mask, (0.1, 0.4), 0.3)
    assert not ends[2].any()
    found = p.nn.policy_loss_grad(p.asarray(logits), *arguments, **options)[2]
    want = differences(lambda z: p.nn.policy_loss(p.asarray(z), *arguments, **options)[0].item(), logits)
    # Central differences: third derivatives of order 10 times step^2, rounding over the step.
    np.testing.assert_allclose(p.asnumpy(found), want, atol=1e-8)
    rng = np.random.default_rng(1)
    logits, targets = rng.standard_normal((2, 2, 3, 4)), rng.integers(0, 4, (2, 2, 3))
    reference, mask = -4 * np.ones((2, 2)), rng.random((2, 2, 3)) < 0.8
    options = dict(mask=mask, beta=0.7, smoothing=0.2)
    found = p.nn.preference_loss_grad(p.asarray(logits), targets, reference, **options)[2]
    want = differences(lambda z: p.nn.preference_loss(p.asarray(z), targets, reference, **options)[0].item(), logits)
    np.testing.assert_allclose(p.asnumpy(found), want, atol=1e-8)


def check_edges(backend, dtype):
    """Logits at the ends of the type, targets outside the vocabulary, nothing kept, nothing there."""
    low, inf = np.finfo(dtype).min, np.inf
    logits = np.array([[0, -inf, 1], [low, low, low], [low, 0, low], [-inf, -inf, -inf], [0, inf, 0], [0, np.nan, 0], [1, 2, 3], [1, 2, 3]], dtype)
    targets = np.array([2, 0, 0, 1, 1, 0, 3, -1])
    got = p.asnumpy(p.nn.token_log_probs(p.asarray(logits, backend=backend), targets))
    one = np.finfo(dtype).eps
    np.testing.assert_allclose(got[:2], [1 - np.log(1 + np.e), -np.log(3)], rtol=4 * one)
    assert got[2] == low and np.isnan(got[3:]).all()
    # A forbidden logit has gradient 0; a row without a finite log-probability is NaN, and alone.
    zero = np.zeros(8, dtype)
    found = p.nn.policy_loss_grad(p.asarray(logits, backend=backend), targets, got, zero + 1, mask=np.arange(8) != 2)
    assert np.isnan(found[0].item())
    grad = p.asnumpy(found[2])
    assert grad[0, 1] == 0 and np.isfinite(grad[:3]).all() and np.isnan(grad[3:]).all()
    # Nothing kept: loss 0, gradients 0.
    none = p.nn.policy_loss_grad(p.asarray(logits, backend=backend), targets, zero, zero, mask=zero != 0)
    assert none[0].item() == 0 and not p.asnumpy(none[1]).any() and not p.asnumpy(none[2]).any()
    for rows in ((0,), (0, 3), (2, 0)):
        empty = p.zeros(rows + (5,), dtype=dtype, backend=backend)
        found = p.nn.policy_loss_grad(empty, np.zeros(rows, np.int64), np.zeros(rows, dtype), np.zeros(rows, dtype))
        assert found[0].item() == 0 and found[1].shape == rows and found[2].shape == rows + (5,)
        assert p.nn.token_log_probs(empty, np.zeros(rows, np.int64)).shape == rows
    half = np.log(2.0)
    for pairs, time in ((0, 3), (3, 0)):
        empty = p.zeros((2, pairs, time, 5), dtype=dtype, backend=backend)
        found = p.nn.preference_loss_grad(empty, np.zeros((2, pairs, time), np.int64), np.zeros((2, pairs), dtype))
        assert abs(found[0].item() - (half if pairs else 0)) <= 2 * one and not p.asnumpy(found[1]).any()
    # Far apart: the loss is the margin itself or nothing, with no overflow.
    far = np.array([[500.0], [0.0]], dtype)
    row = p.zeros((2, 1, 1, 2), dtype=dtype, backend=backend)
    one_token = np.zeros((2, 1, 1), np.int64)
    assert abs(p.nn.preference_loss(row, one_token, far, beta=10.0)[0].item() - 5000) <= 5000 * 4 * one
    assert p.nn.preference_loss(row, one_token, -far, beta=10.0)[0].item() == 0


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_edges(numpy_backend, dtype):
    check_edges(numpy_backend, dtype)


def check_impossible_responses(backend, dtype):
    """A forbidden logit as a token of a response: its sum is -inf and the margin infinite; the loss is what its limit is."""
    logits = np.array([[[[0, 1, 2]], [[0, 0, 0]]], [[[1, -np.inf, 0]], [[0, 1, 0]]]], dtype)
    targets = np.array([[[2], [0]], [[1], [1]]])
    reference = np.array([[-1, -1], [-2, -0.5]], dtype)
    one = np.finfo(dtype).eps
    other = 0.1 * ((-np.log(3) + 1) - (1 - np.log(2 + np.e) + 0.5))  # the second pair's margin
    for swap in (False, True):
        z, y, r = (a[::-1].copy() if swap else a for a in (logits, targets, reference))
        sign = -1 if swap else 1
        for smoothing in (0.0, 1.0, 0.25):
            found = p.nn.preference_loss_grad(*put(backend, z, y, r), smoothing=smoothing)
            alone = p.nn.preference_loss(*put(backend, z, y, r), smoothing=smoothing)
            # The side that the impossible response loses costs nothing, the other all there is.
            free = smoothing == (1.0 if swap else 0.0)
            side = sign * other * (-1 if smoothing == 1 else 1)
            want = np.log1p(np.exp(-side)) / 2 if free else np.inf
            for loss in (found[0].item(), alone[0].item()):
                # A margin and a logarithm near 1: some ten roundings.
                assert abs(loss - want) <= 16 * one if free else loss == want
            sums, grad = p.asnumpy(found[1]), p.asnumpy(found[2])
            assert np.isneginf(sums).sum() == 1 and sums[0 if swap else 1, 0] == -np.inf
            # The pair's slope at an infinite margin is beta / pairs times the weight of the side that it loses.
            slope = 0.05 * (-(1 - smoothing) if swap else smoothing)
            for side, weight in enumerate((slope, -slope)):
                share = np.exp(z[side, 0, 0].astype(float))
                want = weight * ((np.arange(3) == y[side, 0, 0]) - share / share.sum())
                np.testing.assert_allclose(grad[side, 0, 0], want, rtol=16 * one, atol=one)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_impossible_responses(numpy_backend, dtype):
    check_impossible_responses(numpy_backend, dtype)


def check_impossible_tokens(backend, dtype, vocab):
    """An action whose logit is -inf: ratio 0, and an infinite KL term where the reference gives it any probability."""
    rng = np.random.default_rng(vocab)
    logits = rng.standard_normal((3, vocab)).astype(dtype)
    logits[1, 0] = -np.inf
    actions, old = np.array([vocab - 1, 0, 0]), np.full(3, -1.5, dtype)
    advantages, reference = np.array([0.5, -1, 2], dtype), np.array([-1, -2, -np.inf], dtype)

    def call(**options):
        found = p.nn.policy_loss_grad(*put(backend, logits, actions, old, advantages), count=1.0, **options)
        assert p.nn.policy_loss(*put(backend, logits, actions, old, advantages), count=1.0, **options)[0].item() == found[0].item()
        return [p.asnumpy(a) for a in found]

    # Not a NaN: the sum over the tokens is that of its terms, the second of which is infinite.
    loss, log_probs, grad = call(reference_log_probs=reference, kl_weight=0.1)
    assert loss == np.inf and log_probs[1] == -np.inf
    assert np.isfinite(grad[[0, 2]]).all() and not np.isfinite(grad[1, 0])
    # The others' gradients are those that they have beside a possible one, and without the KL term the token's ratio is 0:
    # its gradient is, and of its loss only the clipped side is left, 1 - 0.2 times the advantage.
    kept = call(reference_log_probs=reference, kl_weight=0.1, mask=np.array([True, False, True]))
    assert kept[0] == np.inf  # the last token's reference gives it no probability: exp(d) - d - 1 with d = -inf
    np.testing.assert_array_equal(grad[[0, 2]], kept[2][[0, 2]])
    plain, without = call(), call(mask=np.array([True, False, True]))
    assert abs(plain[0] - without[0] - 0.8) <= 64 * np.finfo(dtype).eps * (1 + abs(without[0])) and not plain[2][1].any()
    kept = call(reference_log_probs=reference, kl_weight=0.1, mask=np.array([True, False, False]))
    assert np.isfinite(kept[0])


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("vocab", [2, 40])
def test_impossible_tokens(numpy_backend, vocab, dtype):
    check_impossible_tokens(numpy_backend, dtype, vocab)


def check_near_policies(backend, dtype):
    """The KL term from policies that nearly agree to ones that are far apart, over a vocabulary of one: the log-probability
    is 0, and d the reference's, both exactly."""
    logits, zero = p.asarray(np.ones((1, 1), dtype), backend=backend), np.zeros(1, dtype)
    for size in [*10.0 ** np.arange(-12, 0), 0.3, 0.999, 1.0, 1.001, 1.999, 2.0, 2.001, 3.7, 10.3, 40.7]:
        for d in (dtype(size), dtype(-size)):
            got = p.nn.policy_loss(logits, [0], zero, zero, reference_log_probs=[d], kl_weight=1.0)[0].item()
            # The definition's series in extended precision, from its smallest term.
            wide = training.WIDE(d)
            terms = [wide * wide / 2]
            while abs(terms[-1]) > 1e-25 * abs(terms[0]) or len(terms) < 2 * abs(d):
                terms.append(terms[-1] * wide / (len(terms) + 2))
            want = sum(sorted(terms, key=abs)) if abs(d) < 2 else np.exp(wide) - 1 - wide
            # An exponential of 3 units of rounding, of which the subtractions leave 2.4 times as many; a rounding.
            assert abs(got - want) <= 8 * np.finfo(dtype).eps / 2 * want, (d, got, want)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_near_policies(numpy_backend, dtype):
    check_near_policies(numpy_backend, dtype)


def test_ties_and_broadcast_advantages(numpy_backend):
    # At the ends of the clip the ratio's own side gives the gradient.
    logits = np.log(np.array([[0.5, 0.5]] * 2))
    old = np.log(np.array([0.5, 0.5]))
    for advantage in (1.0, -1.0):
        grad = p.nn.policy_loss_grad(p.asarray(logits), [0, 1], old, [advantage] * 2, clip=0.0)[2]
        np.testing.assert_allclose(p.asnumpy(grad), np.array([[-0.25, 0.25], [0.25, -0.25]]) * advantage, atol=1e-15)
    rng = np.random.default_rng(0)
    logits, actions = p.asarray(rng.standard_normal((3, 4, 5))), rng.integers(0, 5, (3, 4))
    old, each = rng.standard_normal((3, 4)) - 2, rng.standard_normal((3, 1))
    for narrow in (each, each[:1], each[0], 0.25):
        full = np.broadcast_to(narrow, (3, 4)).copy()
        for one, two in zip(p.nn.policy_loss_grad(logits, actions, old, narrow), p.nn.policy_loss_grad(logits, actions, old, full)):
            np.testing.assert_array_equal(p.asnumpy(one), p.asnumpy(two))


def test_refusals(numpy_backend):
    z, y, one = p.zeros((2, 3, 4), dtype="float32"), np.zeros((2, 3), np.int64), np.zeros((2, 3), np.float32)
    f = p.nn.policy_loss
    with pytest.raises(ValueError, match="vocabulary"):
        f(p.zeros((2, 3, 0), dtype="float32"), y, one, one)
    with pytest.raises(ValueError, match="vocabulary"):
        p.nn.token_log_probs(p.zeros((), dtype="float32"), 0)
    for bad in (y[0], np.zeros((2, 3, 1), np.int64)):
        with pytest.raises(ValueError, match="actions"):
            f(z, bad, one, one)
    for bad in (one, p.zeros((2, 3), dtype="uint32"), y > 0):
        with pytest.raises(p.UnsupportedDtypeError, match="actions"):
            f(z, bad, one, one)
    with pytest.raises(ValueError, match="old_log_probs"):
        f(z, y, one[0], one)
    with pytest.raises(p.UnsupportedDtypeError, match="old_log_probs"):
        f(z, y, p.zeros((2, 3), dtype="float64"), one)
    with pytest.raises(p.UnsupportedDtypeError):
        p.nn.token_log_probs(p.zeros((2, 3, 4), dtype="int32"), y)
    with pytest.raises(ValueError, match="broadcast"):
        f(z, y, one, np.zeros((2, 2), np.float32))
    with pytest.raises(ValueError, match="broadcast"):
        f(z, y, one, np.zeros((1, 2, 3), np.float32))
    with pytest.raises(ValueError, match="mask"):
        f(z, y, one, one, mask=np.ones(3, bool))
    with pytest.raises(p.UnsupportedDtypeError, match="mask"):
        f(z, y, one, one, mask=one)
    with pytest.raises(ValueError, match="kl_weight needs"):
        f(z, y, one, one, kl_weight=0.1)
    for name, bad in [("clip", -0.1), ("clip", np.nan), ("kl_weight", -1), ("kl_weight", np.inf), ("count", 0), ("count", np.nan)]:
        with pytest.raises(ValueError, match=name):
            f(z, y, one, one, reference_log_probs=one, **{name: bad})
    g = p.nn.preference_loss
    pair, ref = p.zeros((2, 1, 3, 4), dtype="float32"), np.zeros((2, 1), np.float32)
    labels = np.zeros((2, 1, 3), np.int64)
    with pytest.raises(ValueError, match="pairs"):
        g(p.zeros((3, 1, 3, 4), dtype="float32"), np.zeros((3, 1, 3), np.int64), ref)
    with pytest.raises(ValueError, match="pairs"):
        g(z, y, ref)
    with pytest.raises(ValueError, match="reference"):
        g(pair, labels, ref[0])
    for name, bad in [("beta", np.nan), ("smoothing", -0.1), ("smoothing", 1.5)]:
        with pytest.raises(ValueError, match=name):
            g(pair, labels, ref, **{name: bad})
    for call in (lambda z: f(z, y, one, one)[0], lambda z: p.nn.token_log_probs(z, y)):
        with pytest.raises(NotImplementedError, match="not captured"):
            p.compile(call)(z)
