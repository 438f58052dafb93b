"""The divergence from a teacher's top logits on the device: against the definition over row lengths, lists and
numbers of rows on both sides of every choice of the kernels."""

import numpy as np
import pytest

import openpacho as p
from test_nn_distillation import check, check_edges, check_repeats, inputs
from test_nn_losses import put

pytestmark = pytest.mark.gpu

# Rows shorter than a vector, of part of a team, of whole teams and one more, up to rows that no team holds.
FEW = [(1, 1, 1), (1, 2, 2), (3, 3, 1), (5, 4, 4), (70, 7, 5), (33, 17, 9), (9, 33, 33), (300, 65, 3), (21, 129, 64), (7, 257, 65), (5, 513, 1),
       (6, 1000, 200), (4, 1025, 1000), (3, 2048, 7), (3, 2049, 1024), (3, 4097, 20), (2, 8193, 64), (3, 16385, 129), (2, 32769, 64),
       (2, 65537, 33), (1, 151001, 20)]  # fmt: skip
# Rows enough to fill the chip.
MANY = [(5000, 5, 2), (3000, 40, 40), (1030, 1500, 16), (600, 5000, 64), (270, 40003, 128)]


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rest", [True, False])
@pytest.mark.parametrize("rows,vocab,entries", FEW)
def test_distillation(hip, rows, vocab, entries, rest, dtype):
    print(rows, vocab, entries, rest, dtype, flush=True)
    check(hip, rows, vocab, entries, dtype, seed=rows + vocab, rest=rest)
    check(hip, rows, vocab, entries, dtype, seed=vocab, rest=rest, masked=False, index=np.int32, temperature=1.0, count=7)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rows,vocab,entries", MANY)
def test_distillation_of_many_rows(hip, rows, vocab, entries, dtype):
    print(rows, vocab, entries, dtype, flush=True)
    check(hip, rows, vocab if dtype == np.float32 else (vocab + 1) // 2, entries if dtype == np.float32 else min(entries, vocab // 2), dtype, seed=5)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_edges(hip, dtype):
    check_edges(hip, dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("vocab", [10, 40, 3000, 20000, 90001])
def test_repeats(hip, vocab, dtype):
    print(vocab, dtype, flush=True)
    check_repeats(hip, dtype, vocab)


@pytest.mark.parametrize("rows,vocab", [(700, 18), (300, 5000), (40, 30000), (3, 100003)])
def test_repeated_calls_give_the_same_bits(hip, rows, vocab):
    given = put(hip, *inputs(rows, vocab, 9, np.float32))
    calls = [p.nn.distillation_loss_grad(*given[:4], mask=given[4], temperature=3.0) for _ in range(3)]
    for again in calls[1:]:
        for one, two in zip(again, calls[0]):
            np.testing.assert_array_equal(p.asnumpy(one), p.asnumpy(two))


def test_the_largest_arrays(hip):
    # Nearly 2^31 logits: the last rows have the bits that they have alone.
    rows, vocab, entries, some = 65531, 32769, 5, 150
    z = p.random.default_rng(2, backend=hip).normal(0, 1, (rows, vocab), dtype=np.float32)
    rng = np.random.default_rng(2)
    order, listed = rng.integers(0, vocab, (rows, entries)), rng.standard_normal((rows, entries)).astype(np.float32)
    rest = rng.standard_normal(rows).astype(np.float32)
    end = slice(rows - some, rows)
    last = z[end]
    _, losses, grad = p.nn.distillation_loss_grad(z, order, listed, rest, count=1.0)
    kept, kept_grad = p.asnumpy(losses)[end], grad[end]
    del grad
    _, want, want_grad = p.nn.distillation_loss_grad(last, order[end], listed[end], rest[end], count=1.0)
    np.testing.assert_array_equal(kept, p.asnumpy(want))
    np.testing.assert_array_equal(p.asnumpy(kept_grad), p.asnumpy(want_grad))
    hip.release_cached_memory()


def test_refusals_at_the_library(hip):
    z = p.zeros((4, 8), dtype=np.float32, backend=hip)._data.ptr
    with hip._active():
        for code, index, rows, vocab, entries, temperature, pointer in [
            (1, 2, 1, 4, 1, 1.0, z), (5, 3, 1, 4, 1, 1.0, z), (5, 2, -1, 4, 1, 1.0, z), (5, 2, 1, 0, 1, 1.0, z), (5, 2, 1, 4, 0, 1.0, z),
            (5, 2, 1, 4, 1025, 1.0, z), (5, 2, 1, 4, 1, 0.0, z), (5, 2, 1, 4, 1, float("nan"), z), (5, 2, 1, 4, 1, 1.0, None)]:  # fmt: skip
            with pytest.raises(ValueError):
                hip._call("hp_distillation_loss", code, index, pointer, *[z] * 2, None, None, *[z] * 3, rows, vocab, entries, temperature, 0.0)
