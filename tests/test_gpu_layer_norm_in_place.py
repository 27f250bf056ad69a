"""Layer norm whose output is its input, in every form that rows have: the bits of a call with arrays of their own."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [1, 255, 257, 513, 1025, 2049, 4097, 8195, 16384, 16385, 40003, 300001])
@pytest.mark.parametrize("rows", [1, 37])
def test_in_place(rt, rows, cols):
    from tinyflow_amd import gpu_op, ndarray
    rng = np.random.RandomState(cols)
    x = rng.normal(0.5, 1, (rows, cols)).astype(np.float32)
    gamma, beta = (rng.normal(0, 1, cols).astype(np.float32) for _ in range(2))
    ax, ag, ab, y = (ndarray.array(v, ctx=rt.ctx) for v in (x, gamma, beta, np.full_like(x, 7.25)))
    gpu_op.layer_norm_forward(ax, ag, ab, y, 1e-5, rt.stream)
    np.testing.assert_array_equal(ax.asnumpy(), x)
    gpu_op.layer_norm_forward(ax, ag, ab, ax, 1e-5, rt.stream)
    np.testing.assert_array_equal(ax.asnumpy(), y.asnumpy())
