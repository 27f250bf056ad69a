"""Dropout from a counter: the mask is the published generator's, the values are a product and a sum of fp32."""
import numpy as np
import pytest

import feed_forward_ref as ref

pytestmark = pytest.mark.gpu


def _array(rt, values):
    from tinyflow_amd import ndarray
    return ndarray.array(np.ascontiguousarray(values, np.float32), ctx=rt.ctx)


def _reference(x, dropout, seed, offset):
    scale = np.float32(1) / (np.float32(1) - np.float32(dropout))
    return np.where(ref.kept(x.size, dropout, seed, offset).reshape(x.shape), x * scale, np.float32(0))


@pytest.mark.parametrize("count", [1, 2, 3, 4, 5, 255, 1024, 4095, 4097, 16384, 100003])
@pytest.mark.parametrize("seed,offset", [(0, 0), (7, 3), (2 ** 64 - 1, 2 ** 63 + 5), (1 << 40, 5 << 32)])
@pytest.mark.parametrize("dropout", [0.1, 0.5])
def test_mask_and_values(rt, count, seed, offset, dropout):
    from tinyflow_amd import gpu_op
    rng = np.random.RandomState(count)
    x, r = (rng.normal(0, 1, count).astype(np.float32) for _ in range(2))
    ax, ar, out = _array(rt, x), _array(rt, r), _array(rt, np.full(count, 9.0))
    wanted = _reference(x, dropout, seed, offset)
    gpu_op.counter_dropout(ax, None, out, dropout, seed, offset, rt.stream)
    np.testing.assert_array_equal(out.asnumpy(), wanted)
    gpu_op.counter_dropout(ax, ar, out, dropout, seed, offset, rt.stream)
    # the product's rounding (half a step) may be left out, and the sum's is half a step
    exact = wanted.astype(np.float64) + r
    ref.assert_within(out.asnumpy(), exact, ref.U * (2 * np.abs(wanted) + np.abs(exact)), "with residual")
    dropped = wanted == 0
    np.testing.assert_array_equal(out.asnumpy()[dropped & (x != 0)], r[dropped & (x != 0)])


@pytest.mark.parametrize("dropout", [0.0, 2.0 ** -33, 1e-3, 0.999, 1 - 2.0 ** -24])
def test_the_ends_of_the_probability(rt, dropout):
    from tinyflow_amd import gpu_op
    x = np.random.RandomState(1).normal(0, 1, 50000).astype(np.float32)
    out = _array(rt, np.zeros_like(x))
    gpu_op.counter_dropout(_array(rt, x), None, out, dropout, 99, 1, rt.stream)
    np.testing.assert_array_equal(out.asnumpy(), _reference(x, dropout, 99, 1))


def test_the_mask_of_the_stored_form(rt):
    """A seed below 2^31 at offset 0 drops what dropout_forward drops."""
    from tinyflow_amd import gpu_op
    x = np.random.RandomState(2).normal(0, 1, (31, 77)).astype(np.float32)
    ax, a, b = _array(rt, x), _array(rt, 0 * x), _array(rt, 0 * x)
    desc = gpu_op.get_input_descriptor(x.shape, "NCHW")
    space, listed, wanted = gpu_op.dropout_forward(ax, a, "NCHW", 0.3, 41, desc, rt.cudnn, rt.stream)
    assert wanted == 0
    gpu_op.counter_dropout(ax, None, b, 0.3, 41, 0, rt.stream)
    np.testing.assert_array_equal(a.asnumpy(), b.asnumpy())
    gpu_op.dropout_backward(a, b, space, listed, rt.cudnn, rt.stream)


def test_offsets_and_seeds_give_other_masks(rt):
    from tinyflow_amd import gpu_op
    x = np.ones(4096, np.float32)
    masks = []
    for seed, offset in ((5, 0), (6, 0), (5, 1), (5, 1 << 32), (5 + (1 << 32), 0)):
        out = _array(rt, 0 * x)
        gpu_op.counter_dropout(_array(rt, x), None, out, 0.5, seed, offset, rt.stream)
        masks.append(out.asnumpy() != 0)
    for i, a in enumerate(masks):
        # 4096 fair draws: 8 standard deviations are 256
        assert abs(int(a.sum()) - 2048) <= 256
        for b in masks[:i]:
            assert abs(int((a != b).sum()) - 2048) <= 256


def test_a_dropped_element_is_zero_whatever_it_held(rt):
    from tinyflow_amd import gpu_op
    x = np.full(1000, np.nan, np.float32)
    x[::2] = np.inf
    out = _array(rt, np.ones(1000))
    gpu_op.counter_dropout(_array(rt, x), None, out, 0.4, 3, 4, rt.stream)
    kept = ref.kept(1000, 0.4, 3, 4)
    got = out.asnumpy()
    assert (got[~kept] == 0).all() and not np.isfinite(got[kept]).any()


def test_in_place(rt):
    from tinyflow_amd import gpu_op
    rng = np.random.RandomState(8)
    x, r = (rng.normal(0, 1, 4999).astype(np.float32) for _ in range(2))
    out = _array(rt, x)
    gpu_op.counter_dropout(_array(rt, x), _array(rt, r), out, 0.25, 17, 2, rt.stream)
    for target in ("input", "residual"):
        ax, ar = _array(rt, x), _array(rt, r)
        gpu_op.counter_dropout(ax, ar, ax if target == "input" else ar, 0.25, 17, 2, rt.stream)
        np.testing.assert_array_equal((ax if target == "input" else ar).asnumpy(), out.asnumpy())


def test_nothing(rt):
    from tinyflow_amd import gpu_op
    a = _array(rt, np.zeros((0, 3)))
    gpu_op.counter_dropout(a, None, a, 0.5, 1, 1, rt.stream)
