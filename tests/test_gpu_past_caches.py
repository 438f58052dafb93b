"""Gradients whose arrays pass the last cache are stored past it: they have the bits of a call on some of the rows."""

import numpy as np
import pytest

import openpacho as p
from test_nn_recurrence import put

pytestmark = pytest.mark.gpu
LAST_CACHE = 1 << 28


@pytest.mark.parametrize("channels", [1371, 1372])
def test_residual_norms(hip, channels):
    rows, some = 8200, 37
    assert 6 * 4 * rows * channels > LAST_CACHE > 6 * 4 * some * channels
    rng = np.random.default_rng(channels)
    d_stream, d_normed, x, stream, gate = rng.standard_normal((5, rows, channels), dtype=np.float32)
    weight, post = rng.standard_normal((2, channels), dtype=np.float32)
    found = []
    for part in (slice(None), slice(rows - some, None)):
        given = put(hip, *(v[part] for v in (d_stream, d_normed, x, stream)), weight)
        dx, d_residual, _, _, d_gate = p.nn.residual_norm_grad(*given, post_weight=put(hip, post)[0], gate=put(hip, gate[part])[0])
        found.append([p.asnumpy(v)[-some:] for v in (dx, d_residual, d_gate)])
    for whole, alone in zip(*found):
        assert np.all(np.isfinite(whole))
        np.testing.assert_array_equal(whole, alone)


@pytest.mark.parametrize("channels", [1001, 1004])
def test_convolutions(hip, channels):
    batch, time, taps = 4, 5600, 4
    assert 3 * 4 * batch * time * channels > LAST_CACHE > 3 * 4 * time * channels
    rng = np.random.default_rng(channels)
    d, x = rng.standard_normal((2, batch, time, channels), dtype=np.float32)
    weight = rng.standard_normal((channels, taps), dtype=np.float32)
    lengths = np.array([time, 5, 0, time - 3])
    found = []
    for part in (slice(None), slice(batch - 1, None)):
        given = put(hip, d[part], x[part], weight)
        dx, *_ = p.nn.causal_conv_grad(*given, activation="silu", lengths=put(hip, lengths[part])[0])
        found.append(p.asnumpy(dx)[-1])
    assert np.all(found[0][time - 3 :] == 0) and np.any(found[0] != 0)
    np.testing.assert_array_equal(*found)
