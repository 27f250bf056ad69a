"""Layer norm, the gated feed-forward product and counter dropout without a GPU: their graphs, and what the calls refuse
before they touch the device."""
import ctypes

import numpy as np
import pytest

from tinyflow_amd import autodiff as ad
from tinyflow_amd import gpu_op, ndarray
from tinyflow_amd.TrainExecute import find_siblings


def _sublayer():
    x, y_ = ad.Variable("x"), ad.Placeholder("y_")
    w = {n: ad.Variable(n) for n in ("gamma", "beta", "gate", "up", "down")}
    n = ad.layer_norm_forward_op(x, w["gamma"], w["beta"])
    h = ad.gated_feed_forward(n, w["gate"], w["up"], "gelu")
    out = ad.counter_dropout_op(ad.matmul_op(h, w["down"]), 0.1, residual=x)
    return x, y_, w, out, ad.softmaxcrossentropy_op(out, y_)


def test_backward_nodes_and_their_shapes():
    x, y_, w, out, loss = _sublayer()
    variables = [x] + list(w.values())
    grads = ad.gradients(loss, variables)
    shapes = {x: (6, 8), y_: (6, 8), w["gamma"]: (8,), w["beta"]: (8,), w["gate"]: (8, 12), w["up"]: (8, 12),
              w["down"]: (12, 8)}
    known = dict(shapes)
    for node in ad.find_topo_sort(grads):
        if node not in known:
            known[node] = tuple(node.op.infer_shape(node, [known[i] for i in node.inputs], None))
    assert [known[g] for g in grads] == [shapes[v] for v in variables]
    # the gradient of the stacked projections is never a value of its own
    kinds = [type(n.op) for n in ad.find_topo_sort(grads)]
    assert ad.GatedActivationBackwardOp not in kinds and kinds.count(ad.GatedBackwardOp) == 3


def test_projections_with_another_reader():
    """Then their adjoints are added up, and the gradients are computed from the sum."""
    x, gate, up = ad.Variable("x"), ad.Variable("gate"), ad.Variable("up")
    pre = ad.gated_projection_op(x, gate, up)
    loss = ad.reduce_sum_op(ad.gated_activation_op(pre, "silu")) + ad.reduce_sum_op(pre)
    dx, dgate, dup = ad.gradients(loss, [x, gate, up])
    assert all(g.activation is None and len(g.inputs) == 4 for g in (dx, dgate, dup))


def test_one_call_for_nodes_of_one_kind():
    x, _, w, out, loss = _sublayer()
    order = ad.find_topo_sort(ad.gradients(loss, [x] + list(w.values())))
    siblings = find_siblings(order, set())
    kinds = sorted((type(first.op).__name__, len(members)) for first, members in siblings.items())
    assert kinds == [("GatedBackwardOp", 3), ("GatedProjectionOp", 2), ("LayerNormBackwardOp", 3)]
    at = {n: i for i, n in enumerate(order)}
    for first, members in siblings.items():
        assert members[0] is first and at[first] == min(at[n] for n in members)
        assert all(at[i] < at[first] for n in members for i in n.inputs if i not in members)
    # two products of one input and other weights, or another activation, are calls of their own
    x, a, b, c = (ad.Variable(n) for n in "xabc")
    one, two = ad.gated_feed_forward(x, a, b), ad.gated_feed_forward(x, a, c)
    again = ad.gated_activation_op(one.inputs[0], "gelu")
    siblings = find_siblings(ad.find_topo_sort([one, two, again]), set())
    assert sorted(len(m) for m in siblings.values()) == [2, 2]
    assert not any(again in m for m in siblings.values())


def test_only_wanted_gradients():
    x, _, w, out, loss = _sublayer()
    order = ad.find_topo_sort(ad.gradients(loss, [w["gate"], w["beta"]]))
    assert sum(isinstance(n.op, ad.GatedBackwardOp) for n in order) == 2   # dgate, and dx for beta


def test_infer_shape_refuses():
    x, a, b = (ad.Variable(n) for n in "xab")
    norm, product = ad.layer_norm_forward_op(x, a, b), ad.gated_projection_op(x, a, b)
    for shapes in [((4, 6), (5,), (5,)), ((4, 6), (6,), (5,)), ((4, 6), (6, 1), (6, 1))]:
        with pytest.raises(ValueError):
            norm.op.infer_shape(norm, shapes, None)
    for shapes in [((4, 6), (5, 3), (5, 3)), ((4, 6), (6, 3), (6, 4)), ((2, 4, 6), (6, 3), (6, 3))]:
        with pytest.raises(ValueError):
            product.op.infer_shape(product, shapes, None)


def test_every_evaluation_has_a_mask_of_its_own(monkeypatch):
    calls = []
    monkeypatch.setattr(gpu_op, "counter_dropout", lambda x, r, out, p, seed, offset, stream: calls.append((seed, offset)))
    x = ad.Variable("x")
    node = ad.counter_dropout_op(x, 0.5)
    other = ad.counter_dropout_op(x, 0.5)
    back, = node.op.gradient(node, x)
    for _ in range(2):
        node.op.compute(node, [None], None, None, None, None)
        node.op.compute_again(node, [None], None, None, None, None)
        back.op.compute(back, [None], None, None, None, None)
    assert calls[0] == calls[1] == calls[2] != calls[3] == calls[4] == calls[5]
    assert node.draw[0] != other.draw[0]


# ------------------------------------------------------------------------------- refusals

class _Fake(ndarray.NDArray):
    """An array that a call must refuse before it reads it: its storage is this process's, not the device's."""
    __slots__ = ["keep"]

    def __init__(self, shape, device=True, data=None, dev_id=0):
        room = np.zeros(max(1, min(int(np.prod(shape)), 1 << 16)), np.float32)
        arr = ndarray.DLArray()
        arr.data = data or room.ctypes.data
        arr.ctx = ndarray.gpu(dev_id) if device else ndarray.cpu(0)
        arr.ndim = len(shape)
        extents = (ctypes.c_int64 * max(1, len(shape)))(*shape)
        arr.shape = extents
        super().__init__(ctypes.pointer(arr))
        self.is_freed = True   # not the library's
        self.keep = (room, extents, arr)


def _refused(call, *args):
    with pytest.raises((RuntimeError, AssertionError)):
        call(*args, None)


def test_layer_norm_refuses():
    x, g, y, host = _Fake((4, 6)), _Fake((6,)), _Fake((4, 6)), _Fake((6,), device=False)
    f, b = gpu_op.layer_norm_forward, gpu_op.layer_norm_backward
    short = _Fake((5,))
    _refused(f, x, short, short, y, 1e-5)
    _refused(f, x, g, short, y, 1e-5)
    _refused(f, x, g, _Fake((6,)), _Fake((6, 4)), 1e-5)
    _refused(f, x, g, host, y, 1e-5)
    _refused(f, x, g, _Fake((6,)), y, -1.0)
    _refused(f, x, g, _Fake((6,)), y, float("nan"))
    _refused(f, x, g, _Fake((6,)), _Fake((4, 6), dev_id=1), 1e-5)
    _refused(f, x, g, _Fake((6,)), _Fake((4, 6), data=x.handle.contents.data + 4), 1e-5)   # overlaps, shifted
    _refused(f, x, g, _Fake((6,)), _Fake((4, 6), data=g.handle.contents.data), 1e-5)
    _refused(b, x, g, y, None, None, None, 1e-5)
    _refused(b, x, g, _Fake((4, 5)), _Fake((4, 6)), None, None, 1e-5)
    _refused(b, x, g, y, _Fake((4, 5)), None, None, 1e-5)
    _refused(b, x, g, y, None, short, None, 1e-5)
    _refused(b, x, g, y, None, None, host, 1e-5)
    _refused(b, x, g, y, x, None, None, 1e-5)   # in place
    d = _Fake((6,))
    _refused(b, x, g, y, None, d, d, 1e-5)


def test_gated_feed_forward_refuses():
    f, b = gpu_op.gated_feed_forward, gpu_op.gated_feed_forward_backward
    x, gate, up = _Fake((4, 6)), _Fake((6, 5)), _Fake((6, 5))
    pre, h = _Fake((2, 4, 5)), _Fake((4, 5))
    _refused(f, x, gate, up, None, None, "silu")
    _refused(f, x, gate, up, pre, h, "swish")
    _refused(f, x, gate, _Fake((6, 4)), pre, h, "silu")
    _refused(f, x, _Fake((5, 6)), _Fake((5, 6)), None, _Fake((4, 6)), "silu")
    _refused(f, x, gate, up, _Fake((4, 2, 5)), h, "silu")
    _refused(f, x, gate, up, None, _Fake((5, 4)), "silu")
    _refused(f, _Fake((1, 4, 6)), gate, up, None, h, "silu")
    _refused(f, x, gate, up, None, _Fake((4, 5), device=False), "silu")
    _refused(f, x, gate, _Fake((6, 5), dev_id=1), None, h, "silu")
    _refused(f, x, gate, up, None, _Fake((4, 5), data=x.handle.contents.data), "silu")
    wide = 1 << 28
    _refused(f, _Fake((4, wide)), _Fake((wide, 2)), _Fake((wide, 2)), None, _Fake((4, 2)), "silu")   # 4 GiB
    dx, dw = _Fake((4, 6)), _Fake((6, 5))
    _refused(b, x, gate, up, pre, h, None, None, None, "silu")
    _refused(b, x, gate, up, None, h, dx, None, None, "silu")    # the projections' gradient is stacked
    _refused(b, x, gate, up, pre, pre, dx, None, None, "silu")
    _refused(b, x, gate, up, pre, h, _Fake((6, 4)), None, None, "silu")
    _refused(b, x, gate, up, pre, h, dx, dw, dw, "silu")
    _refused(b, x, gate, up, pre, h, x, None, None, "silu")
    _refused(b, x, gate, up, pre, h, None, gate, None, "silu")


def test_pointwise_calls_refuse():
    pre, h = _Fake((2, 4, 5)), _Fake((4, 5))
    _refused(gpu_op.gated_activation, pre, _Fake((4, 4)), "silu")
    _refused(gpu_op.gated_activation, _Fake((3, 4, 5)), h, "silu")
    _refused(gpu_op.gated_activation, pre, _Fake((4, 5), data=pre.handle.contents.data), "silu")
    _refused(gpu_op.gated_activation, pre, h, "tanh")
    _refused(gpu_op.gated_activation_backward, pre, h, _Fake((4, 5)), "silu")
    _refused(gpu_op.gated_activation_backward, pre, h, _Fake((2, 4, 5), data=pre.handle.contents.data + 4), "silu")


def test_counter_dropout_refuses():
    f = gpu_op.counter_dropout
    x, y = _Fake((4, 6)), _Fake((4, 6))
    for p in (-0.1, 1.0, 1.5, float("nan"), 1 - 2.0 ** -30):   # the last one is 1 in fp32
        _refused(f, x, None, y, p, 1, 1)
    _refused(f, x, None, _Fake((6, 4)), 0.5, 1, 1)
    _refused(f, x, _Fake((4, 5)), y, 0.5, 1, 1)
    _refused(f, x, None, _Fake((4, 6), device=False), 0.5, 1, 1)
    _refused(f, x, None, _Fake((4, 6), data=x.handle.contents.data + 4), 0.5, 1, 1)
    _refused(f, x, _Fake((4, 6), dev_id=1), y, 0.5, 1, 1)
    for seed, offset in ((-1, 0), (2 ** 64, 0), (0, -1), (0, 2 ** 64)):
        _refused(f, x, None, y, 0.5, seed, offset)


def test_more_than_a_launch_can_count_refuses():
    gamma, x = _Fake(((1 << 26) + 1,)), _Fake((1, (1 << 26) + 1))
    _refused(gpu_op.layer_norm_forward, x, gamma, gamma, x, 1e-5)
    x, h, w = _Fake(((1 << 26) + 1, 1)), _Fake(((1 << 26) + 1, 1)), _Fake((1, 1))
    _refused(gpu_op.gated_feed_forward, x, w, w, None, h, "silu")
    x, h, w = _Fake((1, 1)), _Fake((1, (1 << 26) + 1)), _Fake((1, (1 << 26) + 1))
    _refused(gpu_op.gated_feed_forward, x, w, w, None, h, "silu")
    pre, h = _Fake((2, 1 << 33)), _Fake((1 << 33,))
    _refused(gpu_op.gated_activation, pre, h, "silu")
    _refused(gpu_op.gated_activation_backward, pre, h, pre, "silu")
    x = _Fake((1 << 36,))
    _refused(gpu_op.counter_dropout, x, None, x, 0.5, 1, 1)
