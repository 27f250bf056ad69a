"""Norm, rotation and placement of heads, forward and backward, against float64."""
import ctypes

import numpy as np
import pytest

import attention_ref as ref
from parity import stable_seed

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _device(rt, *values):
    from tinyflow_amd import ndarray
    return [None if v is None else ndarray.array(np.ascontiguousarray(v, np.float32), ctx=rt.ctx) for v in values]


def _empty(rt, shape):
    from tinyflow_amd import ndarray
    return ndarray.array(np.full(shape, 7.25, np.float32), ctx=rt.ctx)   # what is not written shows


def _data(rows, heads, dim, seed):
    rng = np.random.RandomState(seed)
    x = (rng.normal(0, 1, (rows, heads, dim)) * np.exp(0.5 * rng.normal(0, 1, dim))).astype(np.float32)
    gamma = (1 + 0.3 * rng.normal(0, 1, dim)).astype(np.float32)
    dy = (1e-2 * rng.normal(0, 1, (rows, heads, dim))).astype(np.float32)
    return x, gamma, dy


def _frequencies(rotary):
    from tinyflow_amd import gpu_op
    return gpu_op.rotary_frequencies(rotary)


def _check(rt, rows, heads, dim, rotary, interleaved, normed, first=0.0, amplitude=1.25):
    """A call of two parts, the second with one head more, both ways."""
    from tinyflow_amd import gpu_op
    f = _frequencies(rotary) if rotary else None
    positions = (first + np.arange(rows)).astype(np.float32)
    ap, af = _device(rt, positions, f)
    fwd, bwd, checks = [], [], []
    for i in range(2):
        n = heads + i
        x, gamma, dy = _data(rows, n, dim, stable_seed((rows, n, dim, i)))
        gamma = gamma if normed else None
        ax, ag, ady = _device(rt, x.reshape(rows, -1), gamma, dy.reshape(rows, -1))
        y, dx = _empty(rt, (rows, n * dim)), _empty(rt, (rows, n * dim))
        dg = _empty(rt, (dim,)) if normed else None
        fwd.append(gpu_op.head_part(ax, ag, y, n, rotate=bool(rotary)))
        bwd.append(gpu_op.head_gradient_part(ax, ag, ady, dx, dg, n, rotate=bool(rotary)))
        want = ref.Heads(x, gamma, positions if rotary else None, f, amplitude, interleaved, EPS)
        checks.append((want, dy, y, dx, dg, (rows, n, dim)))
    gpu_op.head_rotary(fwd, ap, af, amplitude, interleaved, EPS, None, rt.stream)
    assert gpu_op.head_rotary_backward(bwd, ap, af, amplitude, interleaved, EPS, rt.stream) == 0
    for want, dy, y, dx, dg, shape in checks:
        ref.assert_within(y.asnumpy().reshape(shape), want.y, want.y_tol, "y")
        (wx, tx), of_gamma = want.backward(dy)
        ref.assert_within(dx.asnumpy().reshape(shape), wx, tx, "dx")
        if normed:
            ref.assert_within(dg.asnumpy(), *of_gamma, "dgamma")


# head lengths on both sides of every number of lanes, odd ones, and partly rotated ones that end inside a vector
@pytest.mark.parametrize("dim,rotary", [(1, 0), (2, 2), (5, 4), (30, 30), (64, 64), (64, 10), (72, 36), (80, 40), (96, 96), (128, 128),
                                        (129, 128), (200, 6), (256, 256), (257, 250), (512, 512), (513, 2), (1024, 1024), (1023, 1022)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_against_float64(rt, dim, rotary, interleaved):
    for rows, heads in ((1, 1), (37, 3)):
        _check(rt, rows, heads, dim, rotary, interleaved, True)
    _check(rt, 5, 2, dim, rotary, interleaved, False)


@pytest.mark.parametrize("first", [2.0 ** 20, 2.0 ** 24 - 64, -5.0, 0.5])
def test_far_and_fractional_positions(rt, first):
    _check(rt, 33, 2, 64, 64, False, True, first=first)


@pytest.mark.parametrize("rows,heads,dim", [(5000, 5, 40), (9000, 8, 128), (20011, 1, 8)])
def test_many_rows(rt, rows, heads, dim):
    """Several heads share a row's angles, and workgroups take several rows backward."""
    _check(rt, rows, heads, dim, dim // 2 * 2, True, True)


def test_positions_of_a_sequence_repeat(rt):
    from tinyflow_amd import gpu_op
    x, gamma, _ = _data(12, 2, 16, 1)
    f, positions = _frequencies(16), np.arange(4, dtype=np.float32)
    ax, ag, ap, af = _device(rt, x.reshape(3, 4, 2, 16), gamma, positions, f)
    y = _empty(rt, (3, 4, 2, 16))
    gpu_op.head_rotary([gpu_op.head_part(ax, ag, y, 2)], ap, af, 1.0, False, EPS, None, rt.stream)
    want = ref.Heads(x, gamma, np.tile(positions, 3), f, 1.0, False, EPS)
    ref.assert_within(y.asnumpy().reshape(12, 2, 16), want.y, want.y_tol, "y")


@pytest.mark.parametrize("dim", [24, 31])
def test_placed_rows(rt, dim):
    """Slots in any order; slots that are no row of the cache are left out; other rows and sequences stay as they were."""
    from tinyflow_amd import gpu_op
    batch, tokens, heads, capacity = 2, 5, 3, 9
    rotary = dim // 2 * 2
    x, gamma, _ = _data(batch * tokens, heads, dim, 2)
    slots = np.array([[8, 0, -1, 3, 9], [2, np.nan, 1.5, 7, 6]], np.float32)
    f, positions = _frequencies(rotary), np.arange(10, dtype=np.float32)
    ax, ag, ap, af, slot = _device(rt, x.reshape(batch, tokens, -1), gamma, positions, f, slots)
    k, v, q = (_empty(rt, s) for s in ((batch, capacity, heads * dim), (batch, capacity, heads, dim), (batch, tokens, heads * dim)))
    gpu_op.head_rotary([gpu_op.head_part(ax, ag, q, heads), gpu_op.head_part(ax, ag, k, heads, place=True),
                        gpu_op.head_part(ax, None, v, heads, rotate=False, place=True)], ap, af, 1.0, True, EPS, slot, rt.stream)
    want = ref.Heads(x, gamma, positions, f, 1.0, True, EPS)
    y, tol = want.y.reshape(batch, tokens, -1), want.y_tol.reshape(batch, tokens, -1)
    ref.assert_within(q.asnumpy(), y, tol, "q")
    kept = np.full((batch, capacity, heads * dim), 7.25)
    kept_v, kept_tol = kept.copy(), np.zeros_like(kept)
    for b in range(batch):
        for t in range(tokens):
            s = slots[b, t]
            if s >= 0 and s < capacity and s == np.floor(s):
                kept[b, int(s)], kept_tol[b, int(s)], kept_v[b, int(s)] = y[b, t], tol[b, t], x.reshape(batch, tokens, -1)[b, t]
    ref.assert_within(k.asnumpy(), kept, kept_tol, "keys")
    np.testing.assert_array_equal(v.asnumpy().reshape(kept_v.shape), kept_v)


def test_in_place(rt):
    from tinyflow_amd import gpu_op
    x, gamma, dy = _data(40, 3, 70, 3)
    f, positions = _frequencies(64), np.arange(40, dtype=np.float32)
    ax, ag, ady, ap, af = _device(rt, x.reshape(40, -1), gamma, dy.reshape(40, -1), positions, f)
    y, dx, dg, dg2 = (_empty(rt, s) for s in ((40, 210), (40, 210), (70,), (70,)))
    gpu_op.head_rotary([gpu_op.head_part(ax, ag, y, 3)], ap, af, 1.0, False, EPS, None, rt.stream)
    assert gpu_op.head_rotary_backward([gpu_op.head_gradient_part(ax, ag, ady, dx, dg, 3)], ap, af, 1.0, False, EPS, rt.stream) == 0
    assert gpu_op.head_rotary_backward([gpu_op.head_gradient_part(ax, ag, ady, ady, dg2, 3)], ap, af, 1.0, False, EPS, rt.stream) == 0
    gpu_op.head_rotary([gpu_op.head_part(ax, ag, ax, 3)], ap, af, 1.0, False, EPS, None, rt.stream)
    for a, b in ((y, ax), (dx, ady), (dg, dg2)):
        np.testing.assert_array_equal(a.asnumpy(), b.asnumpy())


def test_one_gradient_alone(rt):
    from tinyflow_amd import gpu_op
    x, gamma, dy = _data(300, 4, 48, 4)
    ax, ag, ady = _device(rt, x.reshape(300, -1), gamma, dy.reshape(300, -1))
    both, dx, dg, dg2 = (_empty(rt, s) for s in ((300, 192), (300, 192), (48,), (48,)))
    part = gpu_op.head_gradient_part
    assert gpu_op.head_rotary_backward([part(ax, ag, ady, both, dg, 4, rotate=False)], None, None, 1.0, False, EPS, rt.stream) == 0
    assert gpu_op.head_rotary_backward([part(ax, ag, ady, dx, None, 4, rotate=False)], None, None, 1.0, False, EPS, rt.stream) == 0
    assert gpu_op.head_rotary_backward([part(ax, ag, ady, None, dg2, 4, rotate=False)], None, None, 1.0, False, EPS, rt.stream) == 0
    np.testing.assert_array_equal(both.asnumpy(), dx.asnumpy())
    np.testing.assert_array_equal(dg.asnumpy(), dg2.asnumpy())


def test_no_rows(rt):
    from tinyflow_amd import gpu_op
    x, dx, dg = _empty(rt, (0, 24)), _empty(rt, (0, 24)), _empty(rt, (12,))
    gamma, p, f = _device(rt, np.ones(12), np.zeros(3), _frequencies(12))
    gpu_op.head_rotary([gpu_op.head_part(x, gamma, dx, 2)], p, f, 1.0, False, EPS, None, rt.stream)
    assert gpu_op.head_rotary_backward([gpu_op.head_gradient_part(x, gamma, x, dx, dg, 2)], p, f, 1.0, False, EPS, rt.stream) == 0
    assert not dg.asnumpy().any()


def test_a_head_that_is_not_finite_stays_alone(rt):
    from tinyflow_amd import gpu_op
    x, gamma, dy = _data(6, 3, 40, 5)
    want = ref.Heads(x, gamma, np.arange(6), _frequencies(40), 1.0, False, EPS)
    x[2, 1, 7], x[4, 0, 39] = np.nan, np.inf
    ax, ag, ady, ap, af = _device(rt, x.reshape(6, -1), gamma, dy.reshape(6, -1), np.arange(6), _frequencies(40))
    y, dx = _empty(rt, (6, 120)), _empty(rt, (6, 120))
    gpu_op.head_rotary([gpu_op.head_part(ax, ag, y, 3)], ap, af, 1.0, False, EPS, None, rt.stream)
    assert gpu_op.head_rotary_backward([gpu_op.head_gradient_part(ax, ag, ady, dx, None, 3)], ap, af, 1.0, False, EPS, rt.stream) == 0
    (wx, tx), _ = want.backward(dy)
    fine = np.ones((6, 3), bool)
    fine[2, 1] = fine[4, 0] = False
    for got, value, tol in ((y, want.y, want.y_tol), (dx, wx, tx)):
        got = got.asnumpy().reshape(6, 3, 40)
        ref.assert_within(got[fine], value[fine], tol[fine], "heads beside it")
        assert np.isnan(got[2, 1]).all() and not np.isfinite(got[4, 0]).all()


def test_gradient_against_differences(rt):
    from tinyflow_amd import gpu_op
    x, gamma, w = _data(8, 2, 24, 21)
    f, positions = _frequencies(16), np.arange(8) + 100.0
    ax, ag, aw, ap, af = _device(rt, x.reshape(8, -1), gamma, w.reshape(8, -1), positions, f)
    dx, dg = _empty(rt, (8, 48)), _empty(rt, (24,))
    assert gpu_op.head_rotary_backward([gpu_op.head_gradient_part(ax, ag, aw, dx, dg, 2)], ap, af, 1.5, True, EPS, rt.stream) == 0
    rng = np.random.RandomState(22)
    for got, at in ((dx, 0), (dg, 1)):
        values = [x.astype(np.float64), gamma.astype(np.float64)]
        direction, h = rng.normal(0, 1, values[at].shape), 1e-5
        sides = []
        for sign in (1, -1):
            moved = list(values)
            moved[at] = values[at] + sign * h * direction
            sides.append((ref.Heads(*moved, positions, f, 1.5, True, EPS).y * w).sum())
        change = (sides[0] - sides[1]) / (2 * h)
        grad = got.asnumpy().astype(np.float64).reshape(direction.shape)
        # third-order remainder h^2, and what fp32 leaves off the gradient
        assert abs(change - (grad * direction).sum()) <= 1e-6 * np.abs(grad * direction).sum() + 1e-8


def test_in_a_captured_graph(rt):
    """What takes no scratch replays to the bits of the eager call; a dgamma is refused."""
    import torch
    from tinyflow_amd import gpu_op
    stream = gpu_op.create_cudaStream()
    x, gamma, dy = _data(3, 2, 64, 6)
    ax, ag, ady, ap, af, slot = _device(rt, x.reshape(3, -1), gamma, dy.reshape(3, -1), np.arange(3), _frequencies(64), np.array([[1, 3, 0]]))
    y, cache, dx, dg = (_empty(rt, s) for s in ((3, 128), (1, 4, 128), (3, 128), (64,)))
    part, back = gpu_op.head_part, gpu_op.head_gradient_part

    def calls():
        gpu_op.head_rotary([part(ax, ag, y, 2), part(ax, ag, cache, 2, place=True)], ap, af, 1.0, False, EPS, slot, stream)
        assert gpu_op.head_rotary_backward([back(ax, ag, ady, dx, None, 2)], ap, af, 1.0, False, EPS, stream) == 0
    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(ctypes.cast(stream.contents, ctypes.c_void_p).value)):
        calls()
        with pytest.raises(RuntimeError):
            gpu_op.head_rotary_backward([back(ax, ag, ady, dx, dg, 2)], ap, af, 1.0, False, EPS, stream)
    for replay in range(3):
        ax[:] = _data(3, 2, 64, 10 + replay)[0].reshape(3, -1)
        ap[:] = np.arange(3, dtype=np.float32) + 7 * replay
        slot[:] = np.array([[replay, 3, -1]], np.float32)
        graph.replay()
        torch.cuda.synchronize()
        got = [a.asnumpy() for a in (y, cache, dx)]
        calls()
        for g, a in zip(got, (y, cache, dx)):
            np.testing.assert_array_equal(g, a.asnumpy())
    gpu_op.destroy_cudaStream(stream)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,dim,rotary", [(9, 64, 8), (9, 128, 64), (4100, 128, 32), (3, 256, 248), (5, 512, 8)])
def test_whole_units_partly_rotated(rt, rows, dim, rotary, interleaved):
    _check(rt, rows, 2 if rows < 4000 else 8, dim, rotary, interleaved, True)


@pytest.mark.parametrize("heads,dim", [(17, 64), (18, 40)])
def test_in_place_of_many_rows(rt, heads, dim):
    """Several heads one behind the other in a lane, the last run of them shorter."""
    from tinyflow_amd import gpu_op
    rows = 4001
    x, gamma, dy = _data(rows, heads, dim, 14)
    f, positions = _frequencies(dim), np.arange(rows, dtype=np.float32)
    ax, ag, ady, ap, af = _device(rt, x.reshape(rows, -1), gamma, dy.reshape(rows, -1), positions, f)
    y, dx, dg, dg2 = (_empty(rt, s) for s in ((rows, heads * dim), (rows, heads * dim), (dim,), (dim,)))
    gpu_op.head_rotary([gpu_op.head_part(ax, ag, y, heads)], ap, af, 1.0, False, EPS, None, rt.stream)
    assert gpu_op.head_rotary_backward([gpu_op.head_gradient_part(ax, ag, ady, dx, dg, heads)], ap, af, 1.0, False, EPS, rt.stream) == 0
    assert gpu_op.head_rotary_backward([gpu_op.head_gradient_part(ax, ag, ady, ady, dg2, heads)], ap, af, 1.0, False, EPS, rt.stream) == 0
    gpu_op.head_rotary([gpu_op.head_part(ax, ag, ax, heads)], ap, af, 1.0, False, EPS, None, rt.stream)
    for a, b in ((y, ax), (dx, ady), (dg, dg2)):
        np.testing.assert_array_equal(a.asnumpy(), b.asnumpy())
