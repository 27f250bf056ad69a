"""Layer norm of rows whose mean is far above their spread, of constant rows and of very long ones: the mean's own rounding must
not show beside the spread.

The bound: n is the longest chain of additions of a row's sum, u = 2^-24.  The first mean is off by D = (n + 2) u mean|x|; the
deviations from it are rounded once each, their mean is off by n u of what they are, mean|x - mu| + D, and their squares' by as much of
mean (x - mu)^2 + 2 D^2.  Nothing is off by u |x| itself.
"""
import numpy as np
import pytest

import feed_forward_ref as ref
from parity import stable_seed

pytestmark = pytest.mark.gpu

U = ref.U
EPS = 1e-5


def _chain(cols):
    """In registers 16 values of a lane, 6 steps across a wave, 16 waves; behind that runs of 256 of a lane's values, and those."""
    return 40.0 if cols <= 16384 else 24.0 + min(256, cols / 1024 + 1) + cols / 2 ** 18


class Centred(ref.Norm):
    def __init__(self, x, gamma, beta, eps):
        ref.Norm.__init__(self, x, gamma, beta, eps)
        x = np.asarray(x, np.float64).reshape(-1, x.shape[-1])
        n = self.n = _chain(x.shape[-1])
        mean = x.mean(1, keepdims=True)
        d = np.abs(x - mean)
        v = (d ** 2).mean(1, keepdims=True)
        first = (n + 2) * U * np.abs(x).mean(1, keepdims=True)
        of_s = 0.5 * (n + 6) * U * (v + 2 * first ** 2) / (v + eps) + 6 * U
        self.d_xh = U * self.s * (d + first + (n + 2) * (d.mean(1, keepdims=True) + first) + 2 * first) + np.abs(self.xh) * of_s
        y = self.y.reshape(x.shape)
        self.y_tol = (np.abs(self.gamma) * (self.d_xh + 2 * U * np.abs(self.xh))
                      + 2 * U * (np.abs(self.beta) + np.abs(y))).reshape(self.shape)


def _check(rt, x, seed, backward=True):
    from tinyflow_amd import gpu_op, ndarray
    rng = np.random.RandomState(seed)
    cols = x.shape[-1]
    gamma, beta = (1 + 0.3 * rng.normal(0, 1, cols)).astype(np.float32), (0.2 * rng.normal(0, 1, cols)).astype(np.float32)
    dy = (rng.normal(0, 1, x.shape) * 1e-2).astype(np.float32)
    ax, ag, ab, ad = (ndarray.array(v, ctx=rt.ctx) for v in (x, gamma, beta, dy))
    norm = Centred(x, gamma, beta, EPS)
    out = ndarray.array(np.full(x.shape, 7.25, np.float32), ctx=rt.ctx)
    gpu_op.layer_norm_forward(ax, ag, ab, out, EPS, rt.stream)
    ref.assert_within(out.asnumpy(), norm.y, norm.y_tol, "y")
    if not backward:
        return
    weights = [ndarray.array(np.full(cols, 7.25, np.float32), ctx=rt.ctx) for _ in range(2)]
    assert gpu_op.layer_norm_backward(ax, ag, ad, out, *weights, EPS, rt.stream) == 0
    for what, got, (value, tol) in zip(("dx", "dgamma", "dbeta"), [out] + weights, norm.backward(dy)):
        ref.assert_within(got.asnumpy(), value, tol, what)


COLS = [1, 3, 100, 257, 700, 1025, 1537, 3000, 5000, 12345, 16384, 16385, 40003]


@pytest.mark.parametrize("cols", COLS)
def test_constant_rows(rt, cols):
    values = np.random.RandomState(cols).uniform(0.1, 1000, 40).astype(np.float32)
    values[0] = 777.7
    _check(rt, np.repeat(values[:, None], cols, 1), cols)


@pytest.mark.parametrize("cols", COLS[1:])
@pytest.mark.parametrize("mean", [300.0, -1e5])
def test_means_above_the_spread(rt, cols, mean):
    rng = np.random.RandomState(stable_seed((cols, int(mean))))
    _check(rt, (rng.normal(0, 1, (9, cols)) + mean).astype(np.float32), cols)


def test_a_million_columns_and_more(rt):
    rng = np.random.RandomState(5)
    for cols in ((1 << 20) + 3, (1 << 24) + 5):
        _check(rt, (rng.normal(0, 1, (1, cols)) + 100).astype(np.float32), cols)
    for value in (777.7, 1.1):
        _check(rt, np.full((1, 1 << 26), value, np.float32), 6, backward=False)
