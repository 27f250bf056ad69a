"""Attention, forward and backward, against float64: sizes on both sides of every tile, masks that end anywhere, rows that see nothing."""
import numpy as np
import pytest

import attention_ref as ref
from parity import stable_seed

pytestmark = pytest.mark.gpu


def _device(rt, *values):
    from tinyflow_amd import ndarray
    return [None if v is None else ndarray.array(np.ascontiguousarray(v, np.float32), ctx=rt.ctx) for v in values]


def _empty(rt, shape):
    from tinyflow_amd import ndarray
    return ndarray.array(np.full(shape, 7.25, np.float32), ctx=rt.ctx)   # what is not written shows


def _data(b, tq, tk, h, hk, d, seed):
    rng = np.random.RandomState(seed)

    def normal(*shape):
        return rng.normal(0, 1, shape)
    return [x.astype(np.float32) for x in (1.5 * normal(b, tq, h, d), normal(b, tk, hk, d), normal(b, tk, hk, d) * np.exp(0.5 * normal(hk, d)),
                                           1e-2 * normal(b, tq, h, d) * np.exp(normal(b, tq, 1, 1)))]


def _run(rt, q, k, v, do, spans=None, slopes=None, cap=0.0, causal=False, backward=True):
    """(out, stat, [dq, dk, dv])"""
    from tinyflow_amd import gpu_op
    b, tq, h, d = q.shape
    hk = k.shape[2]
    arrays = _device(rt, q, k, v, spans, slopes)
    out, stat = _empty(rt, q.shape), _empty(rt, (b, h, tq))
    numbers = (b, h, hk, d ** -0.5, cap, causal, rt.stream)
    assert gpu_op.attention_forward(*arrays, out, stat, *numbers) == 0
    if not backward:
        return out.asnumpy(), stat.asnumpy(), None
    grads = [_empty(rt, x.shape) for x in (q, k, v)]
    ado, = _device(rt, do)
    assert gpu_op.attention_backward(*arrays, out, stat, ado, *grads, *numbers) == 0
    return out.asnumpy(), stat.asnumpy(), [g.asnumpy() for g in grads]


def _check(rt, q, k, v, do, spans=None, slopes=None, cap=0.0, causal=False, backward=True):
    out, stat, grads = _run(rt, q, k, v, do, spans, slopes, cap, causal, backward)
    want = ref.Attention(q, k, v, spans, slopes, q.shape[3] ** -0.5, cap, causal)
    ref.assert_within(out, want.out, want.out_tol, "out")
    ref.assert_within(stat, want.stat, want.stat_tol, "statistics")
    if backward:
        for what, got, (value, tol) in zip(("dq", "dk", "dv"), grads, want.backward(out, stat, do)):
            ref.assert_within(got, value, tol, what)
    return out, stat, grads


# one token; one row short of, at and past a tile; fewer keys than queries (whose first see none); a cache
LENGTHS = [(1, 1), (1, 2), (1, 77), (1, 700), (2, 33), (5, 1), (16, 16), (17, 400), (31, 65), (32, 32), (33, 31), (127, 129), (128, 128), (129, 300),
           (260, 257)]


@pytest.mark.parametrize("tq,tk", LENGTHS)
@pytest.mark.parametrize("d", [16, 64, 72, 128])
def test_against_float64(rt, tq, tk, d):
    for causal in (False, True):
        _check(rt, *_data(2, tq, tk, 2, 1, d, stable_seed((tq, tk, d))), causal=causal)


@pytest.mark.parametrize("d", [1, 2, 3, 5, 31, 33, 63, 65, 80, 96, 100, 127, 129, 160, 200, 255, 256])
def test_head_lengths(rt, d):
    for tq, tk in ((3, 50), (40, 70), (150, 140)):
        _check(rt, *_data(1, tq, tk, 2, 2, d, stable_seed((tq, d))), causal=True)


@pytest.mark.parametrize("h,hk", [(1, 1), (4, 4), (6, 3), (8, 2), (7, 1), (32, 1), (40, 1)])
def test_shared_heads(rt, h, hk):
    for tq, tk in ((1, 90), (2, 40), (70, 70)):
        _check(rt, *_data(2, tq, tk, h, hk, 40, stable_seed((h, hk, tq))), causal=True, slopes=2.0 ** -np.arange(1, h + 1))


def _documents(rng, b, t):
    docs = np.zeros((b, t), int)
    for n in range(b):
        docs[n] = np.sort(rng.randint(0, 4, t))
    return docs


@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("tq", [4, 96, 200])
@pytest.mark.parametrize("mask", ["documents", "prefix", "window", "both", "holes"])
def test_masks(rt, mask, tq, cap):
    from tinyflow_amd import gpu_op
    rng = np.random.RandomState(stable_seed((mask, tq)))
    b = 2
    if mask == "documents":
        spans = gpu_op.attention_spans(tq, documents=_documents(rng, b, tq), causal=True)
    elif mask == "prefix":
        spans = gpu_op.attention_spans(tq, causal=True, prefix=[0, tq // 3])
    elif mask == "window":
        spans = gpu_op.attention_spans(tq, window=7)
    elif mask == "both":
        spans = gpu_op.attention_spans(tq, documents=_documents(rng, b, tq))
    else:   # ends anywhere, past both ends, between whole numbers; empty, reversed and NaN ones see nothing
        first = rng.uniform(-5, tq + 5, (b, tq))
        spans = np.stack([first, first + rng.uniform(-3, tq, (b, tq))], 2).astype(np.float32)
        spans[0, 1], spans[1, 2], spans[1, 0] = (np.nan, 5), (0, np.nan), (-np.inf, np.inf)
    _check(rt, *_data(b, tq, tq, 3, 1, 48, stable_seed((mask, tq))), spans=spans, causal=mask == "holes", cap=cap,
           slopes=np.array([0.5, 0.0, 0.03]))


def test_helper_against_masks(rt):
    """attention_spans' intervals by the definitions of its arguments."""
    from tinyflow_amd import gpu_op
    docs = np.array([[3, 3, 3, 1, 1, 3, 3, 3], [0, 1, 1, 1, 1, 1, 1, 2]])
    spans = gpu_op.attention_spans(8, documents=docs, causal=True, prefix=[2, 0], window=3)
    got = ref.seen(2, 8, 8, spans, False)
    for b in range(2):
        starts = [max(j for j in range(i + 1) if j == 0 or docs[b, j] != docs[b, j - 1]) for i in range(8)]
        for i in range(8):
            for j in range(8):
                own = starts[j] == starts[i]
                ahead = j <= i or j < starts[i] + (2, 0)[b]
                assert got[b, i, j] == (own and ahead and j > i - 3), (b, i, j)


@pytest.mark.parametrize("tq", [1, 3, 40, 140])
def test_rows_that_see_nothing(rt, tq):
    """Output 0, statistics -inf, no gradient from them; keys that nothing sees have none."""
    q, k, v, do = _data(2, tq, 60, 2, 1, 24, tq)
    spans = np.zeros((2, tq, 2), np.float32)
    spans[:, ::3, 1] = 40
    spans[1] = 0
    out, stat, (dq, dk, dv) = _check(rt, q, k, v, do, spans=spans)
    assert not out[1].any() and np.isneginf(stat[1]).all() and not dq[1].any() and not dk[1].any() and not dv[1].any()
    assert not dk[0, 40:].any() and not dv[0, 40:].any()


@pytest.mark.parametrize("tq,tk", [(0, 5), (4, 0), (40, 0), (0, 0)])
def test_nothing(rt, tq, tk):
    out, stat, (dq, dk, dv) = _run(rt, *_data(2, tq, tk, 2, 1, 8, 1))
    assert not out.any() and np.isneginf(stat).all() and not dq.any() and not dk.any() and not dv.any()


@pytest.mark.parametrize("tq,tk", [(1, 200), (6, 150), (150, 150), (300, 300)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, np.finfo(np.float32).max])
def test_what_is_not_seen_may_hold_anything(rt, tq, tk, bad):
    """Causal rows, a document that ends inside a tile, a padded tail: keys, values, queries and gradients behind the masks."""
    q, k, v, do = _data(2, tq, tk, 2, 1, 40, 7)
    used = tk - 37
    spans = np.zeros((2, tq, 2), np.float32)
    spans[..., 1] = np.minimum(used, np.arange(tq) + max(1, used - tq))
    spans[1, tq // 2:] = 0     # rows behind the last sequence
    want = ref.Attention(q, k, v, spans, None, 40 ** -0.5)
    clean = _run(rt, q, k, v, do, spans)
    k[:, used:], v[:, used:, :, 3:] = bad, bad
    q[1, tq // 2:], do[1, tq // 2:] = bad, bad
    # keys that only some rows see
    out, stat, grads = _run(rt, q, k, v, do, spans)
    ref.assert_within(out, want.out, want.out_tol, "out")
    ref.assert_within(stat, want.stat, want.stat_tol, "statistics")
    for a, b in zip(grads, clean[2]):
        assert np.isfinite(a).all()
        np.testing.assert_allclose(a, b, rtol=1e-4, atol=1e-5 * np.abs(b).max())


@pytest.mark.parametrize("tq", [6, 200])
def test_what_is_not_finite_reaches_what_sees_it(rt, tq):
    """One key and one value row: rows that see them are not finite, the others are as they were."""
    q, k, v, do = _data(1, tq, tq, 1, 1, 40, 8)
    want = ref.Attention(q, k, v, None, None, 40 ** -0.5, causal=True)
    at = tq // 2
    for which in (k, v):
        kept = which[0, at, 0, 5]
        which[0, at, 0, 5] = np.nan
        out, stat, (dq, dk, dv) = _run(rt, q, k, v, do, causal=True)
        ref.assert_within(out[:, :at], want.out[:, :at], want.out_tol[:, :at], "out")
        assert np.isnan(out[0, at:, 0, 5]).all()
        if which is k:
            assert np.isnan(out[0, at:]).all() and np.isnan(stat[0, 0, at:]).all()
        (value, tol), _, _ = want.backward(want.out, want.stat, do)
        # statistics and outputs that differ by their rounding
        np.testing.assert_allclose(dq[:, :at], value[:, :at], rtol=0, atol=2e-5 * np.abs(value).max())
        assert np.isnan(dq[0, at:]).any(1).any(1).all()
        which[0, at, 0, 5] = kept


@pytest.mark.parametrize("t", [9, 300])
def test_large_scores(rt, t):
    """Differences of scores far past the exponential's range, and a cap that flattens them."""
    q, k, v, do = _data(1, t, t, 2, 2, 64, 9)
    for cap in (0.0, 10.0):
        _check(rt, 30 * q, k, v, do, causal=True, cap=cap)


@pytest.mark.parametrize("t", [5, 260])
def test_unlike_magnitudes(rt, t):
    """Documents whose values and gradients differ by powers of ten."""
    q, k, v, do = _data(2, t, t, 2, 1, 64, 10)
    v[1] *= np.float32(1e-6)
    do[0] *= np.float32(1e-8)
    k[0, :, :, :8] *= np.float32(1e-7)
    _check(rt, q, k, v, do, causal=True)


@pytest.mark.parametrize("tq,tk", [(8, 30), (130, 140)])
def test_each_result_alone_and_the_same_bits_again(rt, tq, tk):
    from tinyflow_amd import gpu_op
    q, k, v, do = _data(2, tq, tk, 4, 2, 48, 11)
    out, stat, grads = _run(rt, q, k, v, do, causal=True)
    a = _device(rt, q, k, v) + [None, None]
    numbers = (2, 4, 2, 48 ** -0.5, 0.0, True, rt.stream)
    alone = _empty(rt, q.shape), _empty(rt, (2, 4, tq))
    assert gpu_op.attention_forward(*a, alone[0], None, *numbers) == 0
    assert gpu_op.attention_forward(*a, None, alone[1], *numbers) == 0
    np.testing.assert_array_equal(alone[0].asnumpy(), out)
    np.testing.assert_array_equal(alone[1].asnumpy(), stat)
    ado, = _device(rt, do)
    for which in range(3):
        g = [None] * 3
        g[which] = _empty(rt, grads[which].shape)
        assert gpu_op.attention_backward(*a, *alone, ado, *g, *numbers) == 0
        np.testing.assert_array_equal(g[which].asnumpy(), grads[which])


def test_gradients_against_differences(rt):
    rng = np.random.RandomState(22)
    q, k, v, w = _data(1, 12, 15, 2, 1, 10, 23)
    slopes = np.array([0.25, 0.1])
    _, _, grads = _check(rt, q, k, v, w, slopes=slopes, cap=4.0, causal=True)
    for at in range(3):
        values = [x.astype(np.float64) for x in (q, k, v)]
        direction, h = rng.normal(0, 1, values[at].shape), 1e-5
        sides = []
        for sign in (1, -1):
            moved = list(values)
            moved[at] = values[at] + sign * h * direction
            sides.append((ref.Attention(*moved, None, slopes, 10 ** -0.5, 4.0, True).out * w).sum())
        change = (sides[0] - sides[1]) / (2 * h)
        grad = grads[at].astype(np.float64)
        # third-order remainder h^2, and what fp32 leaves off the gradient
        assert abs(change - (grad * direction).sum()) <= 2e-6 * np.abs(grad * direction).sum() + 1e-8


@pytest.mark.parametrize("shape", ["flat", "three", "four"])
def test_array_shapes(rt, shape):
    """[rows, heads D], [batch, tokens, heads D] and [batch, tokens, heads, D] are the same memory."""
    from tinyflow_amd import gpu_op
    q, k, v, do = _data(2, 20, 20, 4, 2, 16, 12)
    out, _, _ = _run(rt, q, k, v, do, backward=False)

    def shaped(x):
        return x.reshape({"flat": (40, -1), "three": (2, 20, -1), "four": x.shape}[shape])
    a = _device(rt, shaped(q), shaped(k), shaped(v))
    got = _empty(rt, shaped(q).shape)
    assert gpu_op.attention_forward(*a, None, None, got, None, 2, 4, 2, 0.25, 0.0, False, rt.stream) == 0
    np.testing.assert_array_equal(got.asnumpy().reshape(out.shape), out)


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("tq,tk", [(3, 900), (700, 900), (700, 20)])
def test_each_gradient_alone_in_pieces(rt, monkeypatch, split, tq, tk):
    """One gradient of three, where walks are cut along the keys, the rows or both; an array of another gradient stays as it was."""
    from tinyflow_amd import gpu_op
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    q, k, v, do = _data(2, tq, tk, 2, 1, 80, 15)
    out, stat, grads = _run(rt, q, k, v, do)
    a = _device(rt, q, k, v) + [None, None] + _device(rt, out, stat, do)
    numbers = (2, 2, 1, 80 ** -0.5, 0.0, False, rt.stream)
    for some in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
        g = [_empty(rt, grads[n].shape) if n in some else None for n in range(3)]
        assert gpu_op.attention_backward(*a, *g, *numbers) == 0
        for n in some:
            np.testing.assert_array_equal(g[n].asnumpy(), grads[n])
