"""The losses from logits on the device: against the definitions over row
lengths and numbers on both sides of every choice of the kernels."""

import numpy as np
import pytest

import openpacho as p
from test_nn_losses import check_edges, check_policy, check_preference, policy_inputs, put

pytestmark = pytest.mark.gpu

# Rows shorter than a vector, of part of a team, of whole teams and one more, up to rows that no team holds.
FEW = [(1, 1), (1, 2), (3, 3), (5, 4), (70, 7), (33, 17), (9, 33), (300, 65), (21, 129), (7, 257), (5, 513), (6, 1000), (4, 1025),
       (3, 2048), (3, 2049), (3, 4097), (2, 8192), (2, 8193), (3, 16385), (2, 32769), (2, 65536), (2, 65537), (1, 151001)]  # fmt: skip
# Rows enough to fill the chip.
MANY = [(5000, 3), (20011, 5), (3000, 40), (1500, 700), (1030, 1500), (700, 3001), (600, 5000), (530, 9001), (300, 20001), (270, 40003)]


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rows,vocab", FEW)
def test_policy_loss(hip, rows, vocab, dtype):
    print(rows, vocab, dtype, flush=True)
    check_policy(hip, rows, vocab, dtype, seed=rows + vocab)
    check_policy(hip, rows, vocab, dtype, seed=vocab, masked=False, reference=False, index=np.int32, clip=(0.1, np.inf), count=7)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rows,vocab", MANY)
def test_policy_loss_of_many_rows(hip, rows, vocab, dtype):
    print(rows, vocab, dtype, flush=True)
    if dtype == np.float64:
        vocab = (vocab + 1) // 2
    check_policy(hip, rows, vocab, dtype, seed=5)


# Rows of which a team holds several at a time, and groups of them that the last rows do not fill.
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rows,vocab", [(257, 1), (1000, 12), (511, 30), (2049, 60), (97, 100), (1003, 200), (338, 254), (85, 400), (41, 512)])
def test_policy_loss_of_short_rows(hip, rows, vocab, dtype):
    print(rows, vocab, dtype, flush=True)
    check_policy(hip, rows, vocab, dtype, seed=rows)


def test_more_short_rows_than_one_launch_has_teams(hip):
    rows, vocab = 16384 * 16 + 37, 130
    rng = np.random.default_rng(8)
    z = p.random.default_rng(8, backend=hip).normal(0, 1, (rows, vocab), dtype=np.float32)
    targets = rng.integers(0, vocab, rows)
    mask = rng.random(rows) < 0.7
    wide = p.asnumpy(z).astype(np.float64)
    share = np.exp(wide)
    share /= share.sum(1, keepdims=True)
    at = np.arange(rows)
    logs = np.where(mask, np.log(share[at, targets]), 0)
    # An exponential, a sum of 130 and a logarithm: some 1e-6 of values up to 10.
    np.testing.assert_allclose(p.asnumpy(p.nn.token_log_probs(z, targets, mask=mask)), logs, rtol=1e-6, atol=2e-6)
    _, found, grad = p.nn.policy_loss_grad(z, targets, logs.astype(np.float32), np.ones(rows, np.float32), mask=mask, count=1.0)
    np.testing.assert_allclose(p.asnumpy(found), logs, rtol=1e-6, atol=2e-6)
    want = share * mask[:, None]
    want[at, targets] -= mask
    np.testing.assert_allclose(p.asnumpy(grad), want, rtol=2e-5, atol=1e-6)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("pairs,time,vocab", [(1, 1, 3), (3, 5, 7), (2, 300, 18), (5, 9, 1025), (2, 7, 9001), (1, 3, 70001), (40, 11, 2050)])
def test_preference_loss(hip, pairs, time, vocab, dtype):
    print(pairs, time, vocab, dtype, flush=True)
    check_preference(hip, pairs, time, vocab, dtype, seed=pairs)
    check_preference(hip, pairs, time, vocab, dtype, seed=time, beta=0.5, smoothing=0.1, index=np.int32)


def test_advantages_broadcast(hip):
    rng = np.random.default_rng(0)
    logits, actions = p.asarray(rng.standard_normal((3, 4, 5, 6)), backend=hip), rng.integers(0, 6, (3, 4, 5))
    old = rng.standard_normal((3, 4, 5)) - 2
    for shape in ((3, 4, 5), (3, 4, 1), (3, 1, 1), (1, 4, 1), (4, 5), (5,), (1,), (), (3, 1, 5), (1, 4, 5)):
        narrow = rng.standard_normal(shape)
        full = np.broadcast_to(narrow, (3, 4, 5)).copy()
        for one, two in zip(p.nn.policy_loss_grad(logits, actions, old, narrow), p.nn.policy_loss_grad(logits, actions, old, full)):
            np.testing.assert_array_equal(p.asnumpy(one), p.asnumpy(two))


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_edges(hip, dtype):
    check_edges(hip, dtype)


@pytest.mark.parametrize("vocab", [9, 3000, 33000, 80001])
def test_forbidden_logits_at_the_ends_of_rows(hip, vocab):
    # Whole pieces and vectors of -inf beside others; the type's lowest value.
    rng = np.random.default_rng(vocab)
    z = rng.standard_normal((6, vocab)).astype(np.float32)
    z[0, : vocab // 2], z[1, vocab // 2 :], z[2, :-1], z[3, 1:] = -np.inf, -np.inf, -np.inf, np.finfo(np.float32).min
    z[4, ::3] = -np.inf
    targets = np.array([vocab - 1, 0, vocab - 1, 0, 1, vocab // 2])
    found = p.nn.policy_loss_grad(p.asarray(z, backend=hip), targets, np.zeros(6, np.float32), np.ones(6, np.float32))
    wide = z.astype(np.float64)
    shifted = np.exp(wide - wide.max(1, keepdims=True))
    share = shifted / shifted.sum(1, keepdims=True)
    logs = np.log(share[np.arange(6), targets])
    np.testing.assert_allclose(p.asnumpy(found[1]), logs, rtol=1e-5, atol=1e-6)
    grad = p.asnumpy(found[2])
    assert np.isfinite(grad).all() and not grad[np.isneginf(z)].any()
    assert p.asnumpy(found[1])[2] == 0 and not grad[2].any()


@pytest.mark.parametrize("rows,vocab", [(1030, 4097), (1500, 6000), (4200, 65), (1100, 66000), (40000, 9), (6000, 12500), (6000, 3000)])
def test_more_sums_than_one_launch_adds(hip, rows, vocab):
    # Losses of rows and workgroups beyond what the last workgroup adds, with and without a mask,
    # which every workgroup counts or (the last of these sizes) a launch of its own.
    rng = np.random.default_rng(rows)
    z = p.random.default_rng(3, backend=hip).normal(0, 1, (rows, vocab), dtype=np.float32)
    actions, advantages = rng.integers(0, vocab, rows), rng.standard_normal(rows).astype(np.float32)
    mask = rng.random(rows) < 0.6
    logs = p.asnumpy(p.nn.token_log_probs(z, actions)).astype(np.float64)
    old = (logs + 0.1 * rng.standard_normal(rows)).astype(np.float32)
    ratio = np.exp(logs - old)
    each = -np.minimum(ratio * advantages, np.clip(ratio, 0.8, 1.2) * advantages)
    for kept in (None, mask):
        want = each[mask].mean() if kept is not None else each.mean()
        found = p.nn.policy_loss_grad(z, actions, old, advantages, mask=kept)
        # A mean of terms of size up to 3, each off by some 1e-6 of the log-probability's rounding.
        assert abs(found[0].item() - want) < 5e-6
        assert abs(p.nn.policy_loss(z, actions, old, advantages, mask=kept)[0].item() - want) < 5e-6


def test_repeated_calls_give_the_same_bits(hip):
    for rows, vocab in ((700, 18), (300, 5000), (3, 100003)):
        given = put(hip, *policy_inputs(rows, vocab, np.float32))
        calls = [p.nn.policy_loss_grad(*given[:4], reference_log_probs=given[4], mask=given[5], kl_weight=0.1) for _ in range(3)]
        for again in calls[1:]:
            for one, two in zip(again, calls[0]):
                np.testing.assert_array_equal(p.asnumpy(one), p.asnumpy(two))


def test_refusals_at_the_library(hip):
    z = p.zeros((4, 8), dtype=np.float32, backend=hip)._data.ptr
    with hip._active():
        for code, index, rows, vocab, logits in [(1, 2, 1, 4, z), (5, 3, 1, 4, z), (5, 2, -1, 4, z), (5, 2, 1, 0, z), (5, 2, 1, 4, None)]:
            with pytest.raises(ValueError):
                hip._call("hp_token_log_probs", code, index, logits, z, None, z, rows, vocab)
            with pytest.raises(ValueError):
                hip._call("hp_policy_loss", code, index, logits, *[z] * 3, 1, 1, None, None, z, z, z, rows, vocab, 0.2, 0.2, 0.0, 0.0)
        with pytest.raises(ValueError, match="clip"):
            hip._call("hp_policy_loss", 5, 2, *[z] * 4, 1, 1, None, None, z, z, z, 1, 4, -0.2, 0.2, 0.0, 0.0)
        with pytest.raises(ValueError, match="repeat"):
            hip._call("hp_policy_loss", 5, 2, *[z] * 4, 1, 0, None, None, z, z, z, 1, 4, 0.2, 0.2, 0.0, 0.0)
        with pytest.raises(ValueError):
            hip._call("hp_preference_loss", 5, 2, *[z] * 3, None, z, z, z, -1, 1, 4, 0.1, 0.0)
        with pytest.raises(ValueError):
            hip._call("hp_preference_loss", 5, 2, None, *[z] * 2, None, z, z, z, 1, 1, 4, 0.1, 0.0)
