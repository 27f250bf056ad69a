"""The gradients of layer norm's weights over so many long rows that one grid dimension would pass 2^32 lanes."""
import numpy as np
import pytest

import feed_forward_ref as ref
from test_gpu_wide_offsets import _over, room  # noqa: F401

pytestmark = pytest.mark.gpu


def test_long_rows_past_one_grid_dimension(rt, room):  # noqa: F811
    """The input is its own output gradient, which one array then holds.  Rows of zeros but for some on either side of 2^22."""
    import torch
    from tinyflow_amd import gpu_op, ndarray
    rows, cols = (1 << 22) + 3, 16385
    picked = [0, 1, 1 << 21, (1 << 22) - 1, 1 << 22, rows - 1]
    x = np.random.RandomState(1).normal(0.3, 1, (len(picked), cols)).astype(np.float32)
    t = room(rows * cols, True).view(rows, cols)
    t[torch.tensor(picked, device="cuda")] = torch.from_numpy(x).cuda()
    torch.cuda.synchronize()
    whole = _over(t, (rows, cols))
    gamma = np.ones(cols, np.float32)
    ag, dgamma, dbeta = (ndarray.array(v, ctx=rt.ctx) for v in (gamma, gamma, gamma))
    assert gpu_op.layer_norm_backward(whole, ag, whole, None, dgamma, dbeta, 1e-5, rt.stream) == 0
    _, *weights = ref.Norm(x, gamma, gamma, 1e-5).backward(x)
    for got, (value, tol), what in zip((dgamma, dbeta), weights, ("dgamma", "dbeta")):
        ref.assert_within(got.asnumpy(), value, tol, what)


@pytest.mark.parametrize("cols", [(1 << 26) - 31, 1 << 26])
def test_gradients_of_the_most_columns_there_are(rt, cols):
    """Both weights' gradients of 2^26 columns are added up by 2^32 lanes.  Of one row they are dy xh and dy."""
    from tinyflow_amd import gpu_op, ndarray
    rng = np.random.RandomState(2)
    x = np.tile(rng.normal(0, 1, 1 << 16).astype(np.float32), cols // (1 << 16) + 1)[:cols][None]
    dy = np.roll(x, 12345, 1)
    ones = np.ones(cols, np.float32)
    ax, ag, ad, dx, dgamma, dbeta = (ndarray.array(v, ctx=rt.ctx) for v in (x, ones, dy, x, ones, ones))
    assert gpu_op.layer_norm_backward(ax, ag, ad, dx, dgamma, dbeta, 1e-5, rt.stream) == 0
    np.testing.assert_array_equal(dbeta.asnumpy(), dy[0])
    mean, square = x.mean(dtype=np.float64), np.dot(x[0, :1 << 16].astype(np.float64), x[0, :1 << 16]) / (1 << 16)
    xh = (x[0] - np.float32(mean)) / np.float32(np.sqrt(square - mean ** 2 + 1e-5))
    # the reference's own roundings, 2^-24 each, and a chain of 256 + 256 + 24 of the squares' sum
    got = dgamma.asnumpy()
    assert (np.abs(got - dy[0] * xh) <= ref.U * (600 * np.abs(dy[0] * xh) + 600 * np.abs(dy[0]))).all()
