"""The gated product where the elements of one sum are of unlike magnitudes: a reduction element far above the others on one side
and zero on the other takes no bits from them.

The bound: an fp32 product's, and what the split on pairs leaves off, 2^-50 of a row's largest value where that is more than
2^-23 of the element."""
import numpy as np
import pytest

import feed_forward_ref as ref

pytestmark = pytest.mark.gpu

U = ref.U


def _arrays(rt, *values):
    from tinyflow_amd import ndarray
    return [ndarray.array(np.ascontiguousarray(v, np.float32), ctx=rt.ctx) for v in values]


def product(a, b):
    """a b and its bound."""
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    A, B = np.abs(a), np.abs(b)
    # two numbers of an element leave 2 u of it off on either side, their smaller ones' product 4 u: half of the 16
    tol = U * (a.shape[1] / 8 + 16) * (A @ B)
    for p, q in ((A, B), (B.T, A.T)):
        off = 2.0 ** -50 * p.max(1, keepdims=True) @ q.sum(0)[None]
        tol = tol + (off if p is A else off.T)
    return a @ b, tol


def _unlike(rng, shape, axis, at, ratio):
    v = rng.normal(0, 1, shape)
    index = [slice(None)] * 2
    index[axis] = at
    v[tuple(index)] *= ratio
    return v.astype(np.float32)


@pytest.mark.parametrize("m,k,f", [(24, 300, 520), (200, 131, 2501), (1100, 1030, 700), (4100, 520, 300)])
@pytest.mark.parametrize("power", [20, 26, 30, 36])
def test_forward(rt, m, k, f, power):
    from tinyflow_amd import gpu_op
    rng = np.random.RandomState(power)
    at = k // 3
    x = _unlike(rng, (m, k), 1, at, 2.0 ** power)
    gate, up = (rng.normal(0, 1, (k, f)).astype(np.float32) for _ in range(2))
    gate[at], up[at] = 0, 0
    pre = _arrays(rt, np.full((2, m, f), 7.25))[0]
    assert gpu_op.gated_feed_forward(*_arrays(rt, x, gate, up), pre, None, "relu", rt.stream) == 0
    for got, w, what in zip(pre.asnumpy(), (gate, up), "gu"):
        ref.assert_within(got, *product(x, w), what)


@pytest.mark.parametrize("m,k,f", [(24, 300, 520), (700, 520, 1000), (4100, 200, 520)])
@pytest.mark.parametrize("power", [20, 26, 30, 36])
def test_backward(rt, m, k, f, power):
    """Columns of the projections' gradients against zero columns of the weights, rows of the input against zero rows of the
    gradients."""
    from tinyflow_amd import gpu_op
    rng = np.random.RandomState(power)
    row, col = m // 3, f // 3
    x = _unlike(rng, (m, k), 0, row, 2.0 ** power)
    d = np.stack([_unlike(rng, (m, f), 1, col, 2.0 ** power) for _ in range(2)])
    gate, up = (rng.normal(0, 1, (k, f)).astype(np.float32) for _ in range(2))
    d[:, row], gate[:, col], up[:, col] = 0, 0, 0
    out = _arrays(rt, *(np.full(v.shape, 7.25) for v in (x, gate, up)))
    ax, ag, au, ad = _arrays(rt, x, gate, up, d)
    assert gpu_op.gated_feed_forward_backward(ax, ag, au, None, ad, *out, "relu", rt.stream) == 0
    wanted = [product(np.concatenate(list(d), 1), np.concatenate([gate, up], 1).T), product(x.T, d[0]), product(x.T, d[1])]
    for got, (value, tol), what in zip(out, wanted, ("dx", "dgate", "dup")):
        ref.assert_within(got.asnumpy(), value, tol, what)
