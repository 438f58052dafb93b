"""``nn.adamw`` on the NumPy backend: steps against the definition, 8-bit moments
against a search for the nearest code, states as values, and what it refuses."""

import numpy as np
import pytest

import openpacho as p
from openpacho.backends import NumpyBackend
from oracle import training

OPTIONS = dict(learning_rate=3e-3, betas=(0.9, 0.99), eps=1e-8)
SHAPES = [(3,), (), (16, 17), (0, 4), (256,), (257,), (1024,), (5, 5, 41), (1,), (2100,)]


def make(shapes, dtype, seed=0):
    rng = np.random.default_rng(seed)

    def normal(shape, scale):
        return np.asarray(scale * rng.standard_normal(shape) * np.exp(2 * rng.standard_normal(shape))).astype(dtype)

    return [[f(shape) for shape in shapes] for f in (
        lambda s: normal(s, 0.1), lambda s: normal(s, 1e-2), lambda s: normal(s, 3e-3), lambda s: np.square(normal(s, 1e-2)))]  # fmt: skip


def put(backend, arrays):
    return [p.asarray(a, backend=backend) for a in arrays]


def bring(arrays):
    return [p.asnumpy(a) for a in arrays]


def near(got, want, units, dtype):
    assert got.dtype == dtype and got.shape == np.shape(want)
    bound = units * np.finfo(dtype).eps / 2 + np.finfo(dtype).tiny
    error = np.abs(got.astype(training.WIDE) - want)
    assert np.all(error <= bound), float(np.max(error / bound))


def check_steps(backend, shapes, dtype, bits=None, seed=0, decays=0.1, count=3):
    given, grads, first, second = make(shapes, dtype, seed)
    params = put(backend, given)
    state = p.nn.adamw_state(params, state_bits=bits, steps=4, first=put(backend, first), second=put(backend, second))
    assert state.steps == 4 and state.state_bits == bits
    each = decays if isinstance(decays, list) else [decays] * len(shapes)
    b1, b2 = OPTIONS["betas"]
    for step in range(count):
        grads = [np.roll(g, 1) for g in grads]
        p0, m0, v0 = bring(params), bring(state.first), bring(state.second)
        if bits and not step:
            for a, b, one, two in zip(m0, v0, first, second):
                if a.size:
                    np.testing.assert_array_equal(a, training.held_first(one))
                    np.testing.assert_array_equal(b, training.held_second(two))
        new, after = p.nn.adamw(params, put(backend, grads), state, weight_decay=decays, **OPTIONS)
        p1, m1, v1 = bring(new), bring(after.first), bring(after.second)
        for i in range(len(shapes)):
            want, units = training.adamw(p0[i], grads[i], m0[i], v0[i], 5 + step, *OPTIONS.values(), each[i])
            near(p1[i], want[0], units[0], dtype)
            if not bits:
                near(m1[i], want[1], units[1], dtype)
                near(v1[i], want[2], units[2], dtype)
            elif grads[i].size:
                # The moments in float32, each operation rounded by itself, and then the nearest codes.
                f = np.float32
                np.testing.assert_array_equal(m1[i], training.held_first(m0[i] * f(b1) + grads[i] * f(1 - b1)))
                np.testing.assert_array_equal(v1[i], training.held_second(v0[i] * f(b2) + grads[i] * grads[i] * f(1 - b2)))
        # What went in is as it was.
        for before, now in zip((p0, m0, v0), (params, state.first, state.second)):
            for a, b in zip(before, bring(now)):
                np.testing.assert_array_equal(a, b)
        assert after.steps == state.steps + 1
        params, state = new, after
    return params, state


@pytest.mark.parametrize("dtype,bits", [(np.float32, None), (np.float64, None), (np.float32, 8)])
def test_steps(numpy_backend, dtype, bits):
    check_steps(numpy_backend, SHAPES, dtype, bits)
    check_steps(numpy_backend, SHAPES, dtype, bits, seed=1, decays=[0.01 * i for i in range(len(SHAPES))])


def check_first_step(backend, dtype):
    """From no moments the first step moves by the learning rate against the gradient's sign."""
    given = np.array([1.0, -2.0, 3.0, 0.5], dtype)
    grad = np.array([0.5, -0.25, 1e-3, 0.0], dtype)
    params = put(backend, [given])
    new, state = p.nn.adamw(params, put(backend, [grad]), p.nn.adamw_state(params), learning_rate=0.5, weight_decay=0)
    np.testing.assert_allclose(bring(new)[0], given - 0.5 * np.sign(grad), rtol=2e-5)
    assert state.steps == 1


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_first_step(numpy_backend, dtype):
    check_first_step(numpy_backend, dtype)


def check_ends(backend, dtype):
    """Gradients whose squares leave the type, and none at all: finite parameters wherever the definition has them."""
    big = np.sqrt(float(np.finfo(dtype).max)) * 10
    given = np.array([1.0, 1.0, 1.0, 1.0, 1.0, 1.0], dtype)
    grad = np.array([0.0, big, -big, 1.0, np.nan, 1e-30], dtype)
    params = put(backend, [given])
    new, state = p.nn.adamw(params, put(backend, [grad]), p.nn.adamw_state(params), learning_rate=0.5, weight_decay=0)
    got, second = bring(new)[0], bring(state.second)[0]
    # An infinite second moment moves nothing; no gradient moves nothing; eps bounds the step of a tiny one.
    assert list(got[:3]) == [1, 1, 1] and np.isinf(second[1:3]).all() and np.isnan(got[4])
    assert abs(got[3] - 0.5) < 1e-4 and abs(got[5] - 1) < 1e-6


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_ends_of_the_type(numpy_backend, dtype):
    check_ends(numpy_backend, dtype)


def check_codes(backend):
    """Every share that has a code, the middles between them, and blocks at the ends of the type."""
    m_grid, u_grid = training._grid(112, 10), training._grid(240, 18)
    for grid, which in ((m_grid, 0), (u_grid, 1)):
        middles = (grid[1:] + grid[:-1]) / 2
        for scale in (1.0, 3.7, 1e-18, 1e18):
            values = np.concatenate([grid, middles, np.nextafter(middles, 0), np.nextafter(middles, 2)]).astype(np.float32)
            for start in range(0, len(values), 255):  # each block led by its largest
                part = np.float32(scale) * np.concatenate([[1], values[start : start + 255]]).astype(np.float32)
                moments = [part, np.square(part) if which else np.zeros_like(part)]
                if which:
                    moments[0] = np.zeros_like(part)
                params = put(backend, [part])
                state = p.nn.adamw_state(params, state_bits=8, first=put(backend, moments[:1]), second=put(backend, moments[1:]))
                np.testing.assert_array_equal(bring(state.first)[0], training.held_first(moments[0]))
                np.testing.assert_array_equal(bring(state.second)[0], training.held_second(moments[1]))
                again = p.nn.adamw_state(params, state_bits=8, first=state.first, second=state.second)
                np.testing.assert_array_equal(bring(again.first)[0], bring(state.first)[0])
                np.testing.assert_array_equal(bring(again.second)[0], bring(state.second)[0])
    tiny, huge = np.finfo(np.float32).smallest_subnormal, np.finfo(np.float32).max
    blocks = [np.zeros(256), np.full(256, tiny), np.full(256, huge), np.full(256, -0.0), np.linspace(0, 1, 256), np.full(256, np.inf),
              np.full(256, 0.5)]  # fmt: skip
    blocks[4][7], blocks[6][200] = 1e-12, np.nan
    given = np.concatenate(blocks).astype(np.float32)
    state = p.nn.adamw_state(put(backend, [given]), state_bits=8, first=put(backend, [-given]), second=put(backend, [given]))
    first, second = bring(state.first)[0], bring(state.second)[0]
    np.testing.assert_array_equal(first, training.held_first(-given))
    np.testing.assert_array_equal(second, training.held_second(given))
    # A moment that is not finite spoils its block and no other; a positive second moment stays positive.
    assert np.isnan(first[5 * 256 :]).all() and np.isfinite(first[: 5 * 256]).all()
    assert (second[4 * 256 : 5 * 256][given[4 * 256 : 5 * 256] > 0] > 0).all()


def test_codes(numpy_backend):
    check_codes(numpy_backend)


def check_resume(backend, bits):
    """A state that is taken up again from its moments goes on with the same bits."""
    given, grads, _, _ = make(SHAPES, np.float32, 3)
    params, grads = put(backend, given), put(backend, grads)
    state = p.nn.adamw_state(params, state_bits=bits)
    for _ in range(3):
        params, state = p.nn.adamw(params, grads, state, **OPTIONS)
    saved = [bring(x) for x in (params, state.first, state.second)]
    again = [put(backend, x) for x in saved]
    resumed = p.nn.adamw_state(again[0], state_bits=bits, steps=state.steps, first=again[1], second=again[2])
    one, state = p.nn.adamw(params, grads, state, **OPTIONS)
    two, resumed = p.nn.adamw(again[0], grads, resumed, **OPTIONS)
    for a, b in ((one, two), (state.first, resumed.first), (state.second, resumed.second)):
        for x, y in zip(bring(a), bring(b)):
            np.testing.assert_array_equal(x, y)


@pytest.mark.parametrize("bits", [None, 8])
def test_resume(numpy_backend, bits):
    check_resume(numpy_backend, bits)


def check_mixed_lists(backend):
    """Lists that hold the state's tensors and others besides, which are of another dtype or backend, wherever these stand."""
    other = NumpyBackend()

    def tensor(size, dtype="float32", where=backend):
        return p.zeros((size,), dtype=dtype, backend=where)

    params = [tensor(3), tensor(2)]
    state = p.nn.adamw_state(params)
    for foreign, error in [(tensor(3, "float64"), p.UnsupportedDtypeError), (tensor(7, "float64"), p.UnsupportedDtypeError),
                           (tensor(3, where=other), p.BackendMismatchError)]:  # fmt: skip
        for at in range(3):
            mixed = params[:at] + [foreign] + params[at:]
            for bad in (mixed, tuple(mixed)):
                with pytest.raises(error):
                    p.nn.adamw(bad, params, state)
                with pytest.raises(error):
                    p.nn.adamw(params, bad, state)
                with pytest.raises(error):
                    p.nn.adamw_state(params, first=bad, second=params)
                with pytest.raises(error):
                    p.nn.adamw_state(params, first=params, second=bad)
        for at in range(2):
            mixed = params[:at] + [foreign] + params[at + 1 :]
            with pytest.raises(error):
                p.nn.adamw(params, mixed, state)
    with pytest.raises(TypeError):
        p.nn.adamw(params, [*params, None], state)


def test_mixed_lists(numpy_backend):
    check_mixed_lists(numpy_backend)


def test_refusals(numpy_backend):
    one, two = p.zeros((3,), dtype="float32"), p.zeros((2, 2), dtype="float32")
    params = [one, two]
    state = p.nn.adamw_state(params)
    with pytest.raises(ValueError, match="no tensors"):
        p.nn.adamw_state([])
    for bad in (one, [np.zeros(3, np.float32)], {"a": one}):
        with pytest.raises(TypeError):
            p.nn.adamw_state(bad)
    with pytest.raises(TypeError):
        p.nn.adamw(params, params, None)
    with pytest.raises(TypeError):
        p.nn.adamw(params, one, state)
    for bad in (params[:1], params[::-1], params + [one]):
        with pytest.raises(ValueError, match="shapes"):
            p.nn.adamw(params, bad, state)
        with pytest.raises(ValueError, match="shapes"):
            p.nn.adamw(bad, params, state)
    wide = [p.zeros(a.shape, dtype="float64") for a in params]
    for bad in (wide, [one, p.zeros((2, 2), dtype="float64")]):
        with pytest.raises(p.UnsupportedDtypeError):
            p.nn.adamw(params, bad, state)
    with pytest.raises(p.UnsupportedDtypeError):
        p.nn.adamw_state([p.zeros((3,), dtype="int32")])
    with pytest.raises(p.UnsupportedDtypeError, match="8 bits"):
        p.nn.adamw_state(wide, state_bits=8)
    for bad in (4, 32, "8"):
        with pytest.raises(ValueError, match="state_bits"):
            p.nn.adamw_state(params, state_bits=bad)
    with pytest.raises(ValueError, match="steps"):
        p.nn.adamw_state(params, steps=-1)
    with pytest.raises(ValueError, match="together"):
        p.nn.adamw_state(params, first=params)
    for name, bad in [("learning_rate", -1), ("learning_rate", np.nan), ("betas", (1.0, 0.9)), ("betas", (0.9, -0.1)), ("eps", 0), ("eps", 1e-39),
                      ("weight_decay", -1), ("weight_decay", [0.1]), ("weight_decay", [0.1, np.inf])]:  # fmt: skip
        with pytest.raises(ValueError, match=name):
            p.nn.adamw(params, params, state, **{name: bad})
    with pytest.raises(NotImplementedError, match="not captured"):
        p.compile(lambda a: p.nn.adamw_state([a]))(one)
    assert "tensors=2" in repr(state)
