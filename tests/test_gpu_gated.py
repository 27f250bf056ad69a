"""The gated feed-forward product, forward and backward, against float64 and against differences."""
import numpy as np
import pytest

import feed_forward_ref as ref
from parity import stable_seed

pytestmark = pytest.mark.gpu

ACTIVATIONS = ["sigmoid", "relu", "silu", "gelu"]
# (rows, width, inner): single tokens and few of them, sizes around every tile's edge, ragged ones, long reductions
SIZES = [(1, 1, 1), (1, 3, 2), (1, 64, 64), (1, 257, 130), (1, 1024, 301), (2, 100, 4), (3, 33, 31), (4, 128, 256), (5, 300, 97),
         (8, 64, 1030), (9, 40, 65), (16, 515, 72), (17, 96, 129), (31, 70, 33), (32, 256, 128), (33, 31, 200), (63, 65, 64),
         (65, 64, 63), (128, 128, 128), (129, 130, 127), (130, 16, 260), (257, 33, 300), (200, 1000, 1), (300, 272, 520),
         (261, 263, 259), (512, 264, 272), (700, 520, 136)]


def _device(rt, *values):
    from tinyflow_amd import ndarray
    return [ndarray.array(np.ascontiguousarray(v, np.float32), ctx=rt.ctx) for v in values]


def _empty(rt, *shape):
    from tinyflow_amd import ndarray
    return ndarray.array(np.full(shape, 7.25, np.float32), ctx=rt.ctx)


def _data(m, k, f, seed):
    rng = np.random.RandomState(seed)
    x = rng.normal(0, 1, (m, k)) * np.exp(rng.normal(0, 1, (m, 1)))
    w = [rng.normal(0, 1, (k, f)) * np.exp(0.5 * rng.normal(0, 1, (1, f))) / np.sqrt(k) for _ in range(2)]
    dh = rng.normal(0, 1, (m, f)) * np.exp(rng.normal(0, 2, (m, 1))) * 1e-3
    return [v.astype(np.float32) for v in (x, w[0], w[1], dh)]


def _forward(rt, x, gate, up, activation, want=("pre", "h")):
    from tinyflow_amd import gpu_op
    m, f = x.shape[0], gate.shape[1]
    pre = _empty(rt, 2, m, f) if "pre" in want else None
    h = _empty(rt, m, f) if "h" in want else None
    assert gpu_op.gated_feed_forward(*_device(rt, x, gate, up), pre, h, activation, rt.stream) == 0
    return [a.asnumpy() for a in (pre, h) if a is not None]


def _backward(rt, x, gate, up, pre, dh, activation, want=(1, 1, 1)):
    from tinyflow_amd import gpu_op
    out = [_empty(rt, *v.shape) if w else None for v, w in zip((x, gate, up), want)]
    arrays = _device(rt, x, gate, up) + (_device(rt, pre) if pre is not None else [None]) + _device(rt, dh)
    assert gpu_op.gated_feed_forward_backward(*arrays, *out, activation, rt.stream) == 0
    return [a.asnumpy() for a in out if a is not None]


@pytest.mark.parametrize("m,k,f", SIZES)
def test_forward(rt, m, k, f):
    activation = ACTIVATIONS[(m + k + f) % 4]
    x, gate, up, _ = _data(m, k, f, stable_seed((m, k, f)))
    (pre_ref, pre_tol), (h_ref, h_tol) = ref.gated(x, gate, up, activation)
    pre, h = _forward(rt, x, gate, up, activation)
    ref.assert_within(pre, pre_ref, pre_tol, "pre")
    ref.assert_within(h, h_ref, h_tol, "h")
    for want in ("pre", "h"):
        alone, = _forward(rt, x, gate, up, activation, (want,))
        np.testing.assert_array_equal(alone, pre if want == "pre" else h)


@pytest.mark.parametrize("m,k,f", SIZES)
def test_backward(rt, m, k, f):
    activation = ACTIVATIONS[(m + k + f + 1) % 4]
    x, gate, up, dh = _data(m, k, f, stable_seed((m, k, f, 1)))
    pre = np.stack([x @ gate, x @ up])
    dpre, d_dpre = ref.pointwise_gradient(pre, dh, activation)
    got = _backward(rt, x, gate, up, pre, dh, activation)
    for what, a, (value, tol) in zip(("dx", "dgate", "dup"), got, ref.gated_backward(x, gate, up, dpre, d_dpre)):
        ref.assert_within(a, value, tol, what)
    for which in range(3):
        want = [i == which for i in range(3)]
        alone, = _backward(rt, x, gate, up, pre, dh, activation, want)
        np.testing.assert_array_equal(alone, got[which])
    # from the projections' gradients themselves
    given = dpre.astype(np.float32)
    for what, a, (value, tol) in zip(("dx", "dgate", "dup"), _backward(rt, x, gate, up, None, given, activation),
                                     ref.gated_backward(x, gate, up, given.astype(np.float64), np.zeros_like(d_dpre))):
        ref.assert_within(a, value, tol, what + " of dpre")


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("m,k,f", [(3, 40, 37), (40, 48, 130), (280, 260, 264)])
def test_every_activation(rt, activation, m, k, f):
    x, gate, up, dh = _data(m, k, f, 5)
    gate *= 3   # into the activations' bends
    (pre_ref, pre_tol), (h_ref, h_tol) = ref.gated(x, gate, up, activation)
    pre, h = _forward(rt, x, gate, up, activation)
    ref.assert_within(pre, pre_ref, pre_tol, "pre")
    ref.assert_within(h, h_ref, h_tol, "h")
    dpre, d_dpre = ref.pointwise_gradient(pre, dh, activation)
    for what, a, (value, tol) in zip(("dx", "dgate", "dup"), _backward(rt, x, gate, up, pre, dh, activation),
                                     ref.gated_backward(x, gate, up, dpre, d_dpre)):
        ref.assert_within(a, value, tol, what)


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("count", [1, 3, 4, 1023, 5000])
def test_pointwise_calls(rt, activation, count):
    from tinyflow_amd import gpu_op
    rng = np.random.RandomState(count)
    pre = rng.normal(0, 3, (2, count)).astype(np.float32)
    pre[0, :1] = 0
    dh = rng.normal(0, 1, count).astype(np.float32)
    ap, ah, ad, h = *_device(rt, pre, dh), _empty(rt, 2, count), _empty(rt, count)
    gpu_op.gated_activation(ap, h, activation, rt.stream)
    act, _, _ = ref.act_and_slope(pre[0].astype(np.float64), activation)
    d_act = 8 * ref.U * (np.abs(pre[0]) + (activation == "sigmoid"))
    ref.assert_within(h.asnumpy(), act * pre[1], np.abs(pre[1]) * d_act + 4 * ref.U * np.abs(act * pre[1]), "h")
    gpu_op.gated_activation_backward(ap, ah, ad, activation, rt.stream)
    value, tol = ref.pointwise_gradient(pre, dh, activation)
    ref.assert_within(ad.asnumpy(), value, tol, "dpre")
    gpu_op.gated_activation_backward(ap, ah, ap, activation, rt.stream)   # in place
    np.testing.assert_array_equal(ap.asnumpy(), ad.asnumpy())


@pytest.mark.parametrize("m,k,f", [(2, 50, 40), (20, 70, 130), (70, 130, 65), (300, 270, 264)])
def test_rows_that_are_not_finite_stay_alone(rt, m, k, f):
    x, gate, up, _ = _data(m, k, f, 13)
    (pre_ref, pre_tol), (h_ref, h_tol) = ref.gated(x, gate, up, "silu")
    row = m // 2
    x[row, k // 3] = np.nan
    pre, h = _forward(rt, x, gate, up, "silu")
    assert np.isnan(pre[:, row]).all() and np.isnan(h[row]).all()
    others = np.arange(m) != row
    ref.assert_within(pre[:, others], pre_ref[:, others], pre_tol[:, others], "pre")
    ref.assert_within(h[others], h_ref[others], h_tol[others], "h")
    x[row, k // 3] = np.inf   # an infinity keeps its sign from the weight
    pre, _ = _forward(rt, x, gate, up, "silu")
    np.testing.assert_array_equal(pre[:, row], np.stack([np.sign(w[k // 3]) * np.inf for w in (gate, up)]).astype(np.float32))
    ref.assert_within(pre[:, others], pre_ref[:, others], pre_tol[:, others], "pre")


@pytest.mark.parametrize("m,k,f", [(3, 60, 70), (270, 260, 264)])
def test_columns_and_gradients_that_are_not_finite(rt, m, k, f):
    x, gate, up, dh = _data(m, k, f, 17)
    (pre_ref, pre_tol), _ = ref.gated(x, gate, up, "silu")
    bad = gate.copy()
    bad[k // 2, f // 3] = -np.inf
    pre, h = _forward(rt, x, bad, up, "silu")
    others = np.arange(f) != f // 3
    assert np.isinf(pre[0, :, f // 3]).all()
    ref.assert_within(pre[0][:, others], pre_ref[0][:, others], pre_tol[0][:, others], "g")
    ref.assert_within(pre[1], pre_ref[1], pre_tol[1], "u")
    pre32 = np.stack([x @ gate, x @ up])
    dpre, d_dpre = ref.pointwise_gradient(pre32, dh, "silu")
    wanted = ref.gated_backward(x, gate, up, dpre, d_dpre)
    dh[m // 2, f // 3] = np.nan
    dx, dgate, dup = _backward(rt, x, gate, up, pre32, dh, "silu")
    rows = np.arange(m) != m // 2
    assert np.isnan(dx[m // 2]).all() and np.isnan(dgate[:, f // 3]).all() and np.isnan(dup[:, f // 3]).all()
    ref.assert_within(dx[rows], wanted[0][0][rows], wanted[0][1][rows], "dx")
    ref.assert_within(dgate[:, others], wanted[1][0][:, others], wanted[1][1][:, others], "dgate")
    ref.assert_within(dup[:, others], wanted[2][0][:, others], wanted[2][1][:, others], "dup")


@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e15])
@pytest.mark.parametrize("m,k,f", [(4, 80, 90), (280, 272, 264)])
def test_the_ends_of_the_range(rt, m, k, f, scale):
    """Operands far from 1: their product stays in the range, their slices have to as well."""
    x, gate, up, dh = _data(m, k, f, 19)
    x, gate, up = x * np.float32(scale), gate / np.float32(scale), up / np.float32(scale)
    (pre_ref, pre_tol), (h_ref, h_tol) = ref.gated(x, gate, up, "gelu")
    pre, h = _forward(rt, x, gate, up, "gelu")
    ref.assert_within(pre, pre_ref, pre_tol, "pre")
    ref.assert_within(h, h_ref, h_tol, "h")
    dpre, d_dpre = ref.pointwise_gradient(pre, dh, "gelu")
    for what, a, (value, tol) in zip(("dx", "dgate", "dup"), _backward(rt, x, gate, up, pre, dh, "gelu"),
                                     ref.gated_backward(x, gate, up, dpre, d_dpre)):
        ref.assert_within(a, value, tol + 2.0 ** -149, what)   # half a step of a subnormal result


@pytest.mark.parametrize("m,k,f", [(4, 80, 90), (280, 272, 264)])
def test_rows_of_zeros(rt, m, k, f):
    x, gate, up, dh = _data(m, k, f, 23)
    x[1], dh[2], gate[:, 3] = 0, 0, 0
    pre, h = _forward(rt, x, gate, up, "silu")
    assert not pre[:, 1].any() and not pre[0][:, 3].any() and not h[1].any()
    dx, dgate, dup = _backward(rt, x, gate, up, pre, dh, "silu")
    assert not dx[2].any()
    assert np.isfinite(dx).all() and np.isfinite(dgate).all() and np.isfinite(dup).all()


def test_empty_extents(rt):
    for m, k, f in [(0, 5, 6), (4, 0, 6), (4, 5, 0)]:
        x, gate, up, dh = (np.ones(s, np.float32) for s in ((m, k), (k, f), (k, f), (m, f)))
        pre, h = _forward(rt, x, gate, up, "silu")
        assert not pre.any() and not h.any()
        for g in _backward(rt, x, gate, up, np.zeros((2, m, f), np.float32), dh, "silu"):
            assert not g.any()


@pytest.mark.parametrize("m,k,f", [(1, 300, 500), (40, 300, 200), (300, 300, 400)])
def test_the_same_bits_again(rt, m, k, f):
    x, gate, up, dh = _data(m, k, f, 29)
    first = _forward(rt, x, gate, up, "silu")
    back = _backward(rt, x, gate, up, first[0], dh, "silu")
    for _ in range(3):
        for a, b in zip(first + back, _forward(rt, x, gate, up, "silu") + _backward(rt, x, gate, up, first[0], dh, "silu")):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid"])
def test_gradient_against_differences(rt, activation):
    m, k, f = 12, 24, 20
    x, gate, up, w = _data(m, k, f, 31)
    pre, _ = _forward(rt, x, gate, up, activation)
    grads = _backward(rt, x, gate, up, pre, w, activation)
    rng = np.random.RandomState(32)

    def loss(x, gate, up):
        return (ref.act_and_slope(x @ gate, activation)[0] * (x @ up) * w).sum()
    for at in range(3):
        values = [v.astype(np.float64) for v in (x, gate, up)]
        direction, h = rng.normal(0, 1, values[at].shape), 1e-5
        sides = []
        for sign in (1, -1):
            moved = list(values)
            moved[at] = values[at] + sign * h * direction
            sides.append(loss(*moved))
        terms = grads[at].astype(np.float64) * direction
        assert abs((sides[0] - sides[1]) / (2 * h) - terms.sum()) <= 1e-5 * np.abs(terms).sum() + 1e-9


def test_streams_that_hand_their_scratch_on(rt):
    from tinyflow_amd import gpu_op
    other = gpu_op.create_cudaStream()
    m, k, f = 300, 280, 290
    x, gate, up, dh = _data(m, k, f, 37)
    pre, h = _forward(rt, x, gate, up, "silu")
    grads = _backward(rt, x, gate, up, pre, dh, "silu")
    arrays = _device(rt, x, gate, up, pre, dh)
    results = []
    for i in range(6):
        stream = (rt.stream, other)[i % 2]
        out = [_empty(rt, *v.shape) for v in (h, x, gate, up)]
        assert gpu_op.gated_feed_forward(*arrays[:3], None, out[0], "silu", stream) == 0
        assert gpu_op.gated_feed_forward_backward(*arrays, *out[1:], "silu", stream) == 0
        results.append(out)
    for out in results:
        for got, wanted in zip(out, [h] + grads):
            np.testing.assert_array_equal(got.asnumpy(), wanted)
    gpu_op.destroy_cudaStream(other)


def test_no_room_for_scratch(rt):
    """Under a budget that the scratch does not fit, the call says how much it wants and leaves its results as they were."""
    from tinyflow_amd import gpu_op
    m, k, f = 600, 400, 1000
    x, gate, up, dh = _data(m, k, f, 41)
    pre, h = _forward(rt, x, gate, up, "silu")
    grads = _backward(rt, x, gate, up, pre, dh, "silu")
    arrays = _device(rt, x, gate, up, pre, dh)
    out = [_empty(rt, *v.shape) for v in (x, gate, up)]
    used = gpu_op.device_memory_stats()[1]
    try:
        gpu_op.set_device_memory_limit(used + (1 << 16))
        wanted = gpu_op.gated_feed_forward_backward(*arrays, *out, "silu", rt.stream)
        assert wanted > 0
        for a in out:
            assert (a.asnumpy() == np.float32(7.25)).all()
    finally:
        gpu_op.set_device_memory_limit(0)
    assert gpu_op.gated_feed_forward_backward(*arrays, *out, "silu", rt.stream) == 0
    for got, value in zip(out, grads):
        np.testing.assert_array_equal(got.asnumpy(), value)


# ---------------------------------------------------------------- sizes of the forward pass on pairs, and long maxima

# the last three: 64 runs and more of the maxima's rows, of the weights' rows, of both
LARGE = [(1027, 1030, 700), (513, 1000, 1543), (2050, 300, 1100), (4040, 130, 1200), (700, 4100, 400), (4100, 4130, 100)]


@pytest.mark.parametrize("m,k,f", LARGE)
def test_large_forward(rt, m, k, f):
    activation = ACTIVATIONS[(m + k + f) % 4]
    x, gate, up, _ = _data(m, k, f, stable_seed((m, k, f)))
    (pre_ref, pre_tol), (h_ref, h_tol) = ref.gated(x, gate, up, activation)
    pre, h = _forward(rt, x, gate, up, activation)
    ref.assert_within(pre, pre_ref, pre_tol, "pre")
    ref.assert_within(h, h_ref, h_tol, "h")
    for want in ("pre", "h"):
        alone, = _forward(rt, x, gate, up, activation, (want,))
        np.testing.assert_array_equal(alone, pre if want == "pre" else h)


@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_large_forward_of_every_activation(rt, activation):
    x, gate, up, _ = _data(1100, 1030, 700, 6)
    gate *= 3   # into the activations' bends
    (pre_ref, pre_tol), (h_ref, h_tol) = ref.gated(x, gate, up, activation)
    pre, h = _forward(rt, x, gate, up, activation)
    ref.assert_within(pre, pre_ref, pre_tol, "pre")
    ref.assert_within(h, h_ref, h_tol, "h")


def test_large_forward_with_values_that_are_not_finite(rt):
    m, k, f = 1027, 1030, 700
    x, gate, up, _ = _data(m, k, f, 19)
    (pre_ref, pre_tol), (h_ref, h_tol) = ref.gated(x, gate, up, "silu")
    rows = np.ones(m, bool)
    for row, value in ((0, np.nan), (130, np.inf), (m - 1, -np.inf)):
        x[row, k // 3] = value
        rows[row] = False
    cols = np.ones(f, bool)
    cols[[5, f - 1]] = False
    bad = gate.copy()
    bad[k - 1, 5], bad[0, f - 1] = -np.inf, np.nan
    pre, h = _forward(rt, x, bad, up, "silu")
    ref.assert_within(pre[0][np.ix_(rows, cols)], pre_ref[0][np.ix_(rows, cols)], pre_tol[0][np.ix_(rows, cols)], "g")
    ref.assert_within(pre[1][rows], pre_ref[1][rows], pre_tol[1][rows], "u")
    ref.assert_within(h[np.ix_(rows, cols)], h_ref[np.ix_(rows, cols)], h_tol[np.ix_(rows, cols)], "h")
    assert np.isnan(pre[0][:, f - 1]).all() and np.isinf(pre[0][rows, 5]).all() and not np.isfinite(pre[:, ~rows]).any()
    np.testing.assert_array_equal(pre[1, 130], np.sign(up[k // 3]) * np.float32(np.inf))


# workgroups of 64 rows, each with one lane group, one row or one column in its last tile
WIDE = [(70, 40, 8300), (65, 16, 8193), (200, 131, 2501), (640, 33, 1000), (129, 1, 4100), (191, 700, 2999), (927, 34, 2382),
        (600, 256, 2500), (2000, 130, 1030)]   # the last ones: a strip a wave


@pytest.mark.parametrize("m,k,f", WIDE)
def test_workgroups_of_64_rows(rt, m, k, f):
    activation = ACTIVATIONS[(m + k + f) % 4]
    x, gate, up, _ = _data(m, k, f, stable_seed((m, k, f)))
    (pre_ref, pre_tol), (h_ref, h_tol) = ref.gated(x, gate, up, activation)
    pre, h = _forward(rt, x, gate, up, activation)
    ref.assert_within(pre, pre_ref, pre_tol, "pre")
    ref.assert_within(h, h_ref, h_tol, "h")
    for want in ("pre", "h"):
        alone, = _forward(rt, x, gate, up, activation, (want,))
        np.testing.assert_array_equal(alone, pre if want == "pre" else h)


@pytest.mark.parametrize("m,k,f", [(9, 0, 6), (40, 0, 70), (200, 0, 2501)])
def test_no_reduction(rt, m, k, f):
    pre, h = _forward(rt, np.ones((m, k), np.float32), *(np.ones((k, f), np.float32) for _ in range(2)), "sigmoid")
    assert not pre.any() and not h.any()


@pytest.mark.parametrize("m,k,f", [(6, 203, 70), (24, 1000, 300), (40, 3000, 70), (200, 131, 2501), (600, 70, 2500)])
@pytest.mark.parametrize("value", [np.inf, np.nan, 3e38])
def test_values_that_cannot_be_sliced(rt, m, k, f, value):
    """Infinities, NaN and values next to the largest in x and in both weights, at the ends of waves' and workgroups' runs of the
    reduction: each stays in the rows and columns that it is of, with its sign."""
    x, gate, up, _ = _data(m, k, f, stable_seed((m, k, f)))
    x, gate, up = (np.clip(v, -1, 1) for v in (x, gate, up))   # products with the largest stay in the range
    along = sorted({0, 7, 8, 15, 16, k // 4, k // 2 - 1, k // 2, k - 1})
    for i, at in enumerate(along):
        gate[at, (5 * i) % f] = value * (-1) ** i
        up[at, (7 * i + 3) % f] = -value * (-1) ** i
    (pre_ref, pre_tol), _ = ref.gated(x, np.where(np.abs(gate) <= 1, gate, 0), np.where(np.abs(up) <= 1, up, 0), "relu")
    pre, = _forward(rt, x, gate, up, "relu", ("pre",))
    for half, w in enumerate((gate, up)):
        plain = (np.abs(w) <= 1).all(0)
        ref.assert_within(pre[half][:, plain], pre_ref[half][:, plain], pre_tol[half][:, plain], "columns without")
        with np.errstate(all="ignore"):
            wanted = x.astype(np.float64) @ w.astype(np.float64)
        for c in np.flatnonzero(~plain):
            if np.isfinite(value):
                tol = ref.product(x, w[:, c:c + 1])[1]
                ref.assert_within(pre[half][:, c:c + 1], wanted[:, c:c + 1], tol, "columns with")
            else:
                np.testing.assert_array_equal(pre[half][:, c], wanted[:, c].astype(np.float32) if np.isinf(value) else
                                              np.full(m, np.nan, np.float32))


# (700 .. 4100, 200): on pairs, the last ones with 64 runs of maxima and more along rows, along columns, of the weights; (4100, 40)
# .. (129, 4100, 60): in one launch, in pieces; (20, 300, 3000) .. (100, 700, 1500): a tile a wave
@pytest.mark.parametrize("m,k,f", [(700, 520, 1000), (1027, 1030, 700), (513, 1000, 1543), (4100, 200, 520), (130, 330, 8200),
                                   (129, 4100, 600), (4100, 40, 70), (130, 33, 8200), (129, 4100, 60), (20, 300, 3000),
                                   (64, 65, 33), (100, 700, 1500)])
def test_backward_with_long_maxima(rt, m, k, f):
    x, gate, up, dh = _data(m, k, f, stable_seed((m, k, f, 1)))
    dh[m // 2] = 0
    dh[m - 1, f - 1] = np.float32(3e4)   # in the last run of both
    pre = np.stack([x @ gate, x @ up])
    dpre, d_dpre = ref.pointwise_gradient(pre, dh, "silu")
    got = _backward(rt, x, gate, up, pre, dh, "silu")
    wanted = ref.gated_backward(x, gate, up, dpre, d_dpre)
    for what, a, (value, tol) in zip(("dx", "dgate", "dup"), got, wanted):
        ref.assert_within(a, value, tol, what)
    for which in range(3):
        want = [i == which for i in range(3)]
        alone, = _backward(rt, x, gate, up, pre, dh, "silu", want)
        np.testing.assert_array_equal(alone, got[which])
    dh[m - 1, f - 1] = np.inf
    dx, dgate, dup = _backward(rt, x, gate, up, pre, dh, "silu")
    assert not np.isfinite(dx[m - 1]).any() and not np.isfinite(dgate[:, f - 1]).any() and not np.isfinite(dup[:, f - 1]).any()
    ref.assert_within(dx[:m - 1], wanted[0][0][:m - 1], wanted[0][1][:m - 1], "dx")
    ref.assert_within(dgate[:, :f - 1], wanted[1][0][:, :f - 1], wanted[1][1][:, :f - 1], "dgate")
    ref.assert_within(dup[:, :f - 1], wanted[2][0][:, :f - 1], wanted[2][1][:, :f - 1], "dup")


@pytest.mark.parametrize("m,k,f", [(5, 70, 203), (40, 131, 1000), (300, 70, 97), (100, 700, 1500), (700, 520, 1000)])
@pytest.mark.parametrize("value", [np.inf, np.nan])
def test_gradients_of_values_that_are_not_finite(rt, m, k, f, value):
    """In dh, in x and in a weight, at the ends of runs: each stays in the sums that it is a term of."""
    x, gate, up, dh = _data(m, k, f, stable_seed((m, k, f)))
    pre = np.stack([x @ gate, x @ up])
    dpre, d_dpre = ref.pointwise_gradient(pre, dh, "silu")
    wanted = ref.gated_backward(x, gate, up, dpre, d_dpre)
    x, gate, dh = x.copy(), gate.copy(), dh.copy()
    rows, cols = sorted({0, m // 2, m - 1}), sorted({0, 7, 8, f // 2, f - 1})
    for i, c in enumerate(cols):
        dh[rows[i % len(rows)], c] = value * (-1) ** i
    gate[k - 1, f // 3], gate[k // 2, 0] = value, -value
    dx, dgate, dup = _backward(rt, x, gate, up, pre, dh, "silu")
    good_rows, good_cols = np.setdiff1d(np.arange(m), rows), np.setdiff1d(np.arange(f), cols)
    good_k = np.setdiff1d(np.arange(k), [k - 1, k // 2])
    assert not np.isfinite(dx[rows]).any()
    assert not np.isfinite(dgate[:, cols]).any() and not np.isfinite(dup[:, cols]).any()
    at = np.ix_(good_rows, good_k)
    ref.assert_within(dx[at], wanted[0][0][at], wanted[0][1][at], "dx")
    assert not np.isfinite(dx[:, [k - 1, k // 2]]).any()
    for what, got, (v, tol) in (("dgate", dgate, wanted[1]), ("dup", dup, wanted[2])):
        ref.assert_within(got[:, good_cols], v[:, good_cols], tol[:, good_cols], what)


@pytest.mark.parametrize("m,k,f", [(0, 70, 40), (200, 0, 40), (200, 70, 0), (0, 700, 1500), (3, 0, 5), (3, 5, 0)])
def test_backward_of_empty_extents(rt, m, k, f):
    x, gate, up, dh = (np.ones(s, np.float32) for s in ((m, k), (k, f), (k, f), (m, f)))
    for pre in (np.zeros((2, m, f), np.float32), None):
        for g in _backward(rt, x, gate, up, pre, dh if pre is not None else np.zeros((2, m, f), np.float32), "sigmoid"):
            assert not g.any()
