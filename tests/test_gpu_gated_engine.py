"""TINYFLOW_SPLIT=0 keeps the gated product, as every other contraction, on the fp32 instruction."""
import numpy as np
import pytest

import feed_forward_ref as ref
from test_gpu_gated import _backward, _data, _forward

pytestmark = pytest.mark.gpu


def product(a, b):
    """a b, and what the fp32 instruction may be off, which adds two products at a time."""
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return a @ b, ref.U * (a.shape[1] / 2 + 16) * (np.abs(a) @ np.abs(b))


# in pieces, 64 rows a workgroup, a strip a wave; sizes that run on pairs
@pytest.mark.parametrize("m,k,f", [(24, 300, 520), (9, 40, 65), (200, 131, 2501), (927, 34, 2382), (1100, 1030, 700)])
def test_forward(rt, m, k, f, monkeypatch):
    x, gate, up, _ = _data(m, k, f, 3)
    x[:, k // 2] *= 2.0 ** 40
    gate[k // 2], up[k // 2] = 0, 0
    pre, h = _forward(rt, x, gate, up, "silu")
    monkeypatch.setenv("TINYFLOW_SPLIT", "0")
    for _ in range(2):
        exact, exact_h = _forward(rt, x, gate, up, "silu")
        for got, w, what in zip(exact, (gate, up), "gu"):
            ref.assert_within(got, *product(x, w), what)
        np.testing.assert_allclose(exact_h, exact[0] * exact[1] / (1 + np.exp(-exact[0].astype(np.float64))), rtol=1e-4, atol=1e-30)
    assert (pre != exact).any()   # another engine's roundings
    monkeypatch.setenv("TINYFLOW_SPLIT", "1")
    np.testing.assert_array_equal(_forward(rt, x, gate, up, "silu")[0], pre)


# a tile a wave, in pieces, on pairs
@pytest.mark.parametrize("m,k,f", [(24, 300, 520), (64, 65, 33), (130, 33, 8200), (700, 520, 1000)])
def test_backward(rt, m, k, f, monkeypatch):
    x, gate, up, dh = _data(m, k, f, 5)
    x[m // 2] *= 2.0 ** 40
    dh[m // 2] = 0
    pre = np.stack([x @ gate, x @ up])
    d = np.stack([dh, dh[::-1]])
    d[:, m // 2] = 0
    plain = _backward(rt, x, gate, up, None, d, "silu"), _backward(rt, x, gate, up, pre, dh, "silu")
    monkeypatch.setenv("TINYFLOW_SPLIT", "0")
    exact = _backward(rt, x, gate, up, None, d, "silu"), _backward(rt, x, gate, up, pre, dh, "silu")
    wanted = [product(np.concatenate(list(d), 1), np.concatenate([gate, up], 1).T), product(x.T, d[0]), product(x.T, d[1])]
    for got, (value, tol), what in zip(exact[0], wanted, ("dx", "dgate", "dup")):
        ref.assert_within(got, value, tol, what)
    for a, b in zip(plain, exact):
        assert any((p != q).any() for p, q in zip(a, b))


def test_values_that_are_not_finite(rt, monkeypatch):
    monkeypatch.setenv("TINYFLOW_SPLIT", "0")
    x, gate, up, _ = _data(300, 280, 264, 7)
    x[7, 3], gate[5, 9] = np.inf, np.nan
    pre, _ = _forward(rt, x, gate, up, "silu")
    rows, cols = np.arange(300) != 7, np.arange(264) != 9
    assert np.isnan(pre[0][:, 9]).all()
    np.testing.assert_array_equal(pre[1, 7], np.sign(up[3]) * np.float32(np.inf))
    at = np.ix_(rows, cols)
    value, tol = product(x[rows], gate[:, cols])
    ref.assert_within(pre[0][at], value, tol, "g")
