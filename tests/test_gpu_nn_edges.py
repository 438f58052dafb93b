"""Operators of ``nn`` on the device at the ends of what they take."""

import numpy as np
import pytest

import openpacho as p
from oracle import training
from test_nn_adamw import check_mixed_lists
from test_nn_losses import check_impossible_responses, check_impossible_tokens, check_near_policies
from test_nn_recurrence import check_infinite_states

pytestmark = pytest.mark.gpu


def test_mixed_lists(hip):
    check_mixed_lists(hip)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_impossible_responses(hip, dtype):
    check_impossible_responses(hip, dtype)


# Short rows, rows of one workgroup, rows in pieces.
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("vocab", [2, 40, 3000, 70001])
def test_impossible_tokens(hip, vocab, dtype):
    check_impossible_tokens(hip, dtype, vocab)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_near_policies(hip, dtype):
    check_near_policies(hip, dtype)


def test_ratios_of_policies_that_are_far_apart(hip):
    # Two equal logits: log-probabilities of -log 2, whose difference from `old` is no float.
    log_prob, one = -np.log(training.WIDE(2)), np.float32(1)
    unit = np.finfo(np.float32).eps / 2
    logits, zero = p.asarray(np.zeros((1, 2), np.float32), backend=hip), np.zeros(1, np.float32)
    rng = np.random.default_rng(0)
    for other in np.concatenate([rng.uniform(-12, 12, 60), [-80, 80]]).astype(np.float32):
        ratio = np.exp(log_prob - training.WIDE(other))
        loss, _, grad = p.nn.policy_loss_grad(logits, [1], [other], [one], clip=(1.0, np.inf))
        # An exponential (a unit in the last place, two of rounding), its correction and the result's rounding.
        assert abs(loss.item() + ratio) <= 4 * unit * ratio, (other, loss.item(), ratio)
        # Shares of exactly a half: the gradient is the ratio's half, both ways.
        assert np.all(np.abs(p.asnumpy(grad)[0] - [ratio / 2, -ratio / 2]) <= 4 * unit * ratio / 2), other
        apart = training.WIDE(other) - log_prob
        excess = np.exp(apart) - 1 - apart
        loss = p.nn.policy_loss(logits, [1], zero, zero, reference_log_probs=[other], kl_weight=1.0)[0].item()
        # The exponential's, of which the subtractions leave 1.7 times as much, and the rounding.
        assert abs(apart) < 0.5 or abs(loss - excess) <= 8 * unit * excess, (other, loss, excess)


# Rows of one wave, of four, of eight and of two runs of these; tiles in one block and in several of both
# lengths, with heads of a channel, packed ones, and ones of whole waves.
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("resets", [True, False])
@pytest.mark.parametrize("sizes", [(1, 1, 3, 3), (2, 4, 70, 70), (2, 15, 12, 6), (2, 50, 70, 35), (3, 120, 13, 13), (2, 250, 256, 4), (2, 1001, 130, 130),
                                   (1, 3000, 256, 2), (1, 15000, 12, 4), (2, 2500, 1030, 1030)])  # fmt: skip
def test_infinite_states(hip, sizes, resets, dtype):
    print(sizes, resets, dtype, flush=True)
    check_infinite_states(hip, sizes, dtype, resets)


def test_one_row_of_many_equal_pieces(hip):
    # 262143 pieces of 8192 logits with one sum, which a chain of additions would round the same way again and again.
    pieces, rng = 262143, np.random.default_rng(1)
    pattern = (rng.integers(-1024, 1024, 8192) / 256).astype(np.float32)
    logits = p.zeros((pieces, 1), dtype=np.float32, backend=hip) + p.asarray(pattern, backend=hip)
    logits = logits.reshape(1, -1)
    total = np.log(training.WIDE(pieces)) + np.log(np.exp(pattern.astype(training.WIDE)).sum())
    for target in (0, 8191, 2**30 + 70, pieces * 8192 - 1):
        found = p.nn.token_log_probs(logits, [target]).item()
        # Units of rounding: an exponential's 4, a piece's sum of 19 additions one after the other, 6 of the pieces' tree,
        # and 25 of the result and its terms.
        want = pattern[target % 8192] - total
        assert abs(found - want) <= 64 * np.finfo(np.float32).eps / 2, (target, found, want)
    hip.release_cached_memory()


def test_advantages_broadcast_to_no_tokens(hip):
    for whole, shape in [((3, 0, 5), (3, 1, 5)), ((2, 3, 0), (2, 1, 1)), ((0, 3, 4), (1, 3, 1)), ((0, 3, 6), (0, 1, 6)), ((2, 0, 3, 4), (2, 1, 3, 1)),
                         ((2, 0), ()), ((3, 4, 0), (4, 1))]:  # fmt: skip
        logits, advantages = (p.zeros(s, dtype=np.float32, backend=hip) for s in (whole + (6,), shape))
        found = p.nn.policy_loss_grad(logits, np.zeros(whole, np.int64), np.zeros(whole, np.float32), advantages)
        assert found[0].item() == 0 and found[1].shape == whole and found[2].shape == whole + (6,)
