"""Layer norm forward and backward against float64 and against differences, over row lengths on both sides of every
form that the kernels have."""
import numpy as np
import pytest

import feed_forward_ref as ref
from parity import stable_seed

pytestmark = pytest.mark.gpu

EPS = 1e-5
# 1 .. 3: shorter than a vector; 256 .. 16384: ends of the forms in registers; 16385, 40003: rows that do not fit
COLS = [1, 2, 3, 5, 64, 255, 256, 257, 511, 513, 1023, 1024, 1025, 2047, 2049, 4096, 4097, 8192, 8195, 16384, 16385, 40003]


def _device(rt, *values):
    from tinyflow_amd import ndarray
    return [ndarray.array(np.ascontiguousarray(v, np.float32), ctx=rt.ctx) for v in values]


def _empty(rt, shape):
    from tinyflow_amd import ndarray
    return ndarray.array(np.full(shape, 7.25, np.float32), ctx=rt.ctx)   # what is not written shows


def _data(shape, seed, mean=0.3):
    rng = np.random.RandomState(seed)
    cols = shape[-1]
    x = (rng.normal(0, 1, shape) * np.exp(0.5 * rng.normal(0, 1, cols)) + mean).astype(np.float32)
    return (x, (1 + 0.3 * rng.normal(0, 1, cols)).astype(np.float32), (0.2 * rng.normal(0, 1, cols)).astype(np.float32),
            (rng.normal(0, 1, shape) * 1e-2).astype(np.float32))


def _check(rt, shape, x, gamma, beta, dy, eps=EPS):
    from tinyflow_amd import gpu_op
    ax, ag, ab, ady = _device(rt, x, gamma, beta, dy)
    y, dx, dg, db = (_empty(rt, s) for s in (shape, shape, gamma.shape, gamma.shape))
    gpu_op.layer_norm_forward(ax, ag, ab, y, eps, rt.stream)
    assert gpu_op.layer_norm_backward(ax, ag, ady, dx, dg, db, eps, rt.stream) == 0
    norm = ref.Norm(x, gamma, beta, eps)
    ref.assert_within(y.asnumpy(), norm.y, norm.y_tol, "y")
    for what, got, (value, tol) in zip(("dx", "dgamma", "dbeta"), (dx, dg, db), norm.backward(dy)):
        ref.assert_within(got.asnumpy(), value, tol, what)
    np.testing.assert_array_equal(ax.asnumpy(), x)
    return y, dx, dg, db


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("rows", [1, 7, 130])
def test_against_float64(rt, rows, cols):
    if rows * cols > 1 << 20:
        rows = 3
    _check(rt, (rows, cols), *_data((rows, cols), stable_seed((rows, cols))))


@pytest.mark.parametrize("shape", [(5,), (2, 3, 40), (3, 2, 2, 9), (3000, 48), (4100, 257), (1030, 1100)])
def test_ranks_and_many_rows(rt, shape):
    _check(rt, shape, *_data(shape, stable_seed(shape)))


def test_a_mean_far_above_the_spread(rt):
    """The squares are taken behind the mean: no cancellation."""
    _check(rt, (9, 700), *_data((9, 700), 3, mean=1000.0))


def test_values_whose_squares_leave_the_range(rt):
    x, gamma, beta, dy = _data((4, 300), 5)
    _check(rt, (4, 300), x * np.float32(1e-18), gamma, beta, dy)   # variance below eps
    _check(rt, (4, 300), x * np.float32(1e15), gamma, beta, dy)


def test_constant_rows(rt):
    from tinyflow_amd import gpu_op
    x = np.full((3, 640), 2.5, np.float32)
    _, gamma, beta, _ = _data((3, 640), 1)
    ax, ag, ab = _device(rt, x, gamma, beta)
    y = _empty(rt, x.shape)
    gpu_op.layer_norm_forward(ax, ag, ab, y, EPS, rt.stream)
    np.testing.assert_array_equal(y.asnumpy(), np.broadcast_to(beta, x.shape))


@pytest.mark.parametrize("cols", [48, 2000, 20000])
def test_a_row_that_is_not_finite_stays_alone(rt, cols):
    from tinyflow_amd import gpu_op
    x, gamma, beta, dy = _data((6, cols), 11)
    norm = ref.Norm(x, gamma, beta, EPS)
    x[2, 1], x[4, cols - 1] = np.nan, np.inf
    ax, ag, ab, ady = _device(rt, x, gamma, beta, dy)
    y, dx = _empty(rt, x.shape), _empty(rt, x.shape)
    gpu_op.layer_norm_forward(ax, ag, ab, y, EPS, rt.stream)
    assert gpu_op.layer_norm_backward(ax, ag, ady, dx, None, None, EPS, rt.stream) == 0
    others = [0, 1, 3, 5]
    value, tol = norm.backward(dy)[0]
    for got, value, tol in ((y.asnumpy(), norm.y, norm.y_tol), (dx.asnumpy(), value, tol)):
        assert np.isnan(got[[2, 4]]).all()
        ref.assert_within(got[others], value[others], tol[others], "rows beside it")


@pytest.mark.parametrize("cols", [100, 1500, 17000])
def test_each_gradient_alone_and_the_same_bits_again(rt, cols):
    from tinyflow_amd import gpu_op
    shape = (37, cols)
    x, gamma, beta, dy = _data(shape, 4)
    _, *together = _check(rt, shape, x, gamma, beta, dy)
    together = [a.asnumpy() for a in together]
    ax, ag, ady = _device(rt, x, gamma, dy)
    for _ in range(2):
        for which in range(3):
            out = [None] * 3
            out[which] = _empty(rt, together[which].shape)
            assert gpu_op.layer_norm_backward(ax, ag, ady, *out, EPS, rt.stream) == 0
            np.testing.assert_array_equal(out[which].asnumpy(), together[which])


def test_no_rows(rt):
    from tinyflow_amd import gpu_op
    x, dx = _empty(rt, (0, 12)), _empty(rt, (0, 12))
    gamma, beta = _device(rt, np.ones(12), np.ones(12))
    dg, db = _empty(rt, (12,)), _empty(rt, (12,))
    gpu_op.layer_norm_forward(x, gamma, beta, dx, EPS, rt.stream)
    assert gpu_op.layer_norm_backward(x, gamma, x, dx, dg, db, EPS, rt.stream) == 0
    assert not dg.asnumpy().any() and not db.asnumpy().any()


def test_in_place(rt):
    from tinyflow_amd import gpu_op
    for cols in (130, 3000, 20000):
        x, gamma, beta, _ = _data((5, cols), cols)
        ax, ag, ab = _device(rt, x, gamma, beta)
        y = _empty(rt, x.shape)
        gpu_op.layer_norm_forward(ax, ag, ab, y, EPS, rt.stream)
        gpu_op.layer_norm_forward(ax, ag, ab, ax, EPS, rt.stream)
        np.testing.assert_array_equal(ax.asnumpy(), y.asnumpy())


def test_gradient_against_differences(rt):
    """sum(w y) changes by sum(dx dir) h: central differences in float64 of the float64 norm, along random directions."""
    x, gamma, beta, w = _data((8, 96), 21)
    _, dx, dg, db = _check(rt, (8, 96), x, gamma, beta, w)
    rng = np.random.RandomState(22)
    for got, at in ((dx, 0), (dg, 1), (db, 2)):
        values = [x.astype(np.float64), gamma.astype(np.float64), beta.astype(np.float64)]
        direction, h = rng.normal(0, 1, values[at].shape), 1e-5
        sides = []
        for sign in (1, -1):
            moved = list(values)
            moved[at] = values[at] + sign * h * direction
            sides.append((ref.Norm(*moved, EPS).y * w).sum())
        change = (sides[0] - sides[1]) / (2 * h)
        grad = got.asnumpy().astype(np.float64)
        # third-order remainder h^2, and what fp32 leaves off the gradient
        tol = 1e-6 * np.abs(grad * direction).sum() + 1e-8
        assert abs(change - (grad * direction).sum()) <= tol


def test_another_stream_behind_the_first(rt):
    """The gradients' scratch goes from one stream to another."""
    from tinyflow_amd import gpu_op
    shape = (600, 900)
    x, gamma, beta, dy = _data(shape, 9)
    norm = ref.Norm(x, gamma, beta, EPS)
    wanted = norm.backward(dy)
    other = gpu_op.create_cudaStream()
    ax, ag, ady = _device(rt, x, gamma, dy)
    outs = []
    for i in range(6):
        out = [_empty(rt, shape), _empty(rt, gamma.shape), _empty(rt, gamma.shape)]
        assert gpu_op.layer_norm_backward(ax, ag, ady, *out, EPS, (rt.stream, other)[i % 2]) == 0
        outs.append(out)
    for out in outs:
        for got, (value, tol) in zip(out, wanted):
            ref.assert_within(got.asnumpy(), value, tol, "on its stream")
    gpu_op.destroy_cudaStream(other)


def test_more_waves_than_a_grid_dimension_counts(rt):
    """2^26 rows and a wave each pass 2^32 lanes in one dimension: the rows at both ends, and each side of where it wraps."""
    from tinyflow_amd import gpu_op, ndarray
    rows = (1 << 26) + 5
    x = np.empty((rows, 2), np.float32)
    x[:, 0] = np.arange(rows, dtype=np.float32) % 1021 + 1
    x[:, 1] = -x[:, 0]
    ax, ag, ab = _device(rt, x, np.float32([1, 2]), np.float32([0.5, -0.25]))
    y = ndarray.empty(x.shape, ctx=rt.ctx)
    gpu_op.array_set(y, 7.25, rt.stream)   # what is not written shows
    gpu_op.layer_norm_forward(ax, ag, ab, y, 0.0, rt.stream)
    # every row is (v, -v): its mean is 0 and its deviation v, a division and a root off by half a step each, the product by another
    np.testing.assert_allclose(y.asnumpy(), np.broadcast_to(np.float32([1.5, -2.25]), x.shape), rtol=0, atol=2 * 4 * 2.0 ** -24)
    gpu_op.layer_norm_backward(ax, ag, ax, y, None, None, 1e30, rt.stream)
    # an eps of 1e30 makes s = 1e-15 and xh next to nothing: dx = s (a - mean(a)), a = (v, -2 v), so s (1.5 v, -1.5 v)
    s = 1 / np.sqrt(1e30)
    want = (np.float64(1.5 * s) * x).astype(np.float32)
    np.testing.assert_allclose(y.asnumpy(), want, rtol=8 * 2.0 ** -24, atol=0)
