"""The gated product of subnormal operands, whose bits the split has to scale up before it takes them apart."""
import numpy as np
import pytest

import feed_forward_ref as ref
from test_gpu_gated import _backward, _data, _forward

pytestmark = pytest.mark.gpu


# vector multiply-adds; in registers; on pairs
@pytest.mark.parametrize("m,k,f", [(3, 64, 96), (24, 300, 520), (1100, 1030, 700)])
@pytest.mark.parametrize("scale", [1e-38, 1e-41])
def test_forward(rt, m, k, f, scale):
    x, gate, up, _ = _data(m, k, f, 3)
    x, gate, up = x * np.float32(scale), gate * np.float32(1e30), up * np.float32(1e30)
    (pre_ref, pre_tol), _ = ref.gated(x, gate, up, "relu")
    pre, = _forward(rt, x, gate, up, "relu", ("pre",))
    ref.assert_within(pre, pre_ref, pre_tol, "pre")


@pytest.mark.parametrize("m,k,f", [(24, 300, 520), (700, 520, 1000)])
@pytest.mark.parametrize("scale", [1e-38, 1e-41])
def test_backward(rt, m, k, f, scale):
    x, gate, up, dh = _data(m, k, f, 5)
    d = (np.stack([dh, dh[::-1]]) * 1e3).astype(np.float32) * np.float32(scale)
    x, gate, up = (v * np.float32(1e30) for v in (x, gate, up))
    wanted = ref.gated_backward(x, gate, up, d.astype(np.float64), np.zeros(d.shape))
    for got, (value, tol), what in zip(_backward(rt, x, gate, up, None, d, "relu"), wanted, ("dx", "dgate", "dup")):
        ref.assert_within(got, value, tol, what)
