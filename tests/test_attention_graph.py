"""Norm and rotation of heads, and attention, without a GPU: their graphs, the helpers that make their inputs, and what the calls refuse
before they touch the device."""
import ctypes

import numpy as np
import pytest

from test_feed_forward_graph import _Fake, _refused
from tinyflow_amd import autodiff as ad
from tinyflow_amd import gpu_op
from tinyflow_amd.TrainExecute import find_siblings


def _sublayer(masks=True):
    """(x, placeholders, weights, loss) of 2 sequences of 6 tokens, 4 heads of 8 columns over 2, and the shapes of all leaves"""
    x, y_ = ad.Variable("x"), ad.Placeholder("y_")
    w = {n: ad.Variable(n) for n in ("wq", "wk", "wv", "wo", "gq", "gk")}
    fed = {n: ad.Placeholder(n) for n in ("positions", "frequencies", "spans", "slopes")}
    shapes = {x: (12, 10), y_: (12, 10), w["wq"]: (10, 32), w["wk"]: (10, 16), w["wv"]: (10, 16), w["wo"]: (32, 10), w["gq"]: (8,),
              w["gk"]: (8,), fed["positions"]: (6,), fed["frequencies"]: (3,), fed["spans"]: (2, 6, 2), fed["slopes"]: (4,)}
    out = ad.self_attention(x, w["wq"], w["wk"], w["wv"], w["wo"], 2, 4, 2, (w["gq"], w["gk"]), fed["positions"], fed["frequencies"],
                            spans=fed["spans"] if masks else None, slopes=fed["slopes"] if masks else None)
    return x, w, ad.softmaxcrossentropy_op(out + x, y_), shapes


def _infer(nodes, known):
    known = dict(known)
    for node in ad.find_topo_sort(nodes):
        if node not in known:
            known[node] = tuple(node.op.infer_shape(node, [known[i] for i in node.inputs], None))
    return known


@pytest.mark.parametrize("masks", [True, False])
def test_backward_nodes_and_their_shapes(masks):
    x, w, loss, shapes = _sublayer(masks)
    variables = [x] + list(w.values())
    grads = ad.gradients(loss, variables)
    known = _infer(grads, shapes)
    assert [known[g] for g in grads] == [shapes[v] for v in variables]
    kinds = [type(n.op) for n in ad.find_topo_sort(grads)]
    assert kinds.count(ad.AttentionStatisticsOp) == 1 and kinds.count(ad.AttentionBackwardOp) == 3
    assert kinds.count(ad.HeadRotaryBackwardOp) == 4
    statistics, = [n for n in known if isinstance(n.op, ad.AttentionStatisticsOp)]
    assert known[statistics] == (2, 4, 6)


def test_one_call_for_nodes_of_one_kind():
    x, w, loss, _ = _sublayer()
    order = ad.find_topo_sort([loss] + ad.gradients(loss, [x] + list(w.values())))
    siblings = find_siblings(order, set())
    kinds = sorted((tuple(sorted(type(n.op).__name__ for n in members))) for members in siblings.values())
    assert kinds == [("AttentionBackwardOp",) * 3, ("AttentionForwardOp", "AttentionStatisticsOp"), ("HeadRotaryBackwardOp",) * 2,
                     ("HeadRotaryBackwardOp",) * 2]
    at = {n: i for i, n in enumerate(order)}
    for first, members in siblings.items():
        assert members[0] is first and at[first] == min(at[n] for n in members)
        assert all(at[i] < at[first] for n in members for i in n.inputs if i not in members)
    # two attentions of the same inputs under other masks are calls of their own
    q, k, v = (ad.Variable(n) for n in "qkv")
    one, two = ad.attention_forward_op(q, k, v, 1, 2), ad.attention_forward_op(q, k, v, 1, 2, causal=True)
    order = ad.find_topo_sort([one, two, ad.attention_statistics_op(one)])
    (members,) = find_siblings(order, set()).values()
    assert two not in members and len(members) == 2


def test_one_node_as_queries_keys_and_values():
    x = ad.Variable("x")
    dx, = ad.gradients(ad.reduce_sum_op(ad.attention_forward_op(x, x, x, 1, 2)), [x])
    assert _infer([dx], {x: (5, 12)})[dx] == (5, 12)


def test_infer_shape_refuses():
    x, g, p, f = (ad.Variable(n) for n in "xgpf")
    node = ad.head_rotary_op(x, 3, g, p, f)
    assert node.op.infer_shape(node, [(4, 24), (8,), (4,), (4,)], None) == (4, 24)
    for shapes in ([(4, 25), (8,), (4,), (4,)], [(4, 24), (7,), (4,), (4,)], [(4, 24), (8,), (4,), (5,)], [(1, 4, 2, 8), (8,), (4,), (4,)]):
        with pytest.raises(ValueError):
            node.op.infer_shape(node, shapes, None)
    with pytest.raises(ValueError):
        ad.head_rotary_op(x, 3, g, p, None)
    node = ad.attention_forward_op(x, g, p, 2, 4, 2)
    assert node.op.infer_shape(node, [(6, 32), (8, 16), (8, 16)], None) == (6, 32)
    for shapes in ([(6, 32), (8, 16), (8, 32)], [(6, 32), (8, 24), (8, 24)], [(7, 32), (8, 16), (8, 16)], [(6, 33), (8, 16), (8, 16)]):
        with pytest.raises(ValueError):
            node.op.infer_shape(node, shapes, None)


# -------------------------------------------------------------------------------- helpers

def test_frequencies():
    f = gpu_op.rotary_frequencies(8)
    np.testing.assert_allclose(f, 10000.0 ** -np.array([0, 0.25, 0.5, 0.75]), rtol=2.0 ** -24)
    np.testing.assert_allclose(gpu_op.rotary_frequencies(8, factor=4), f / 4, rtol=2.0 ** -23)
    parts = gpu_op.rotary_frequencies(8, factor=4, context=2048)
    assert parts[0] == f[0] and abs(parts[3] / f[3] - 0.25) < 1e-6 and f[2] / 4 < parts[2] < f[2]
    for columns in (0, 3):
        with pytest.raises(ValueError):
            gpu_op.rotary_frequencies(columns)


def test_spans():
    np.testing.assert_array_equal(gpu_op.attention_spans(3), [[0, 3]] * 3)
    np.testing.assert_array_equal(gpu_op.attention_spans(3, causal=True), [[0, 1], [0, 2], [0, 3]])
    np.testing.assert_array_equal(gpu_op.attention_spans(2, 5, window=3), [[1, 4], [2, 5]])
    np.testing.assert_array_equal(gpu_op.attention_spans(2, 9, causal=True, used=[4, 9]), [[[0, 3], [0, 4]], [[0, 8], [0, 9]]])
    np.testing.assert_array_equal(gpu_op.attention_spans(4, causal=True, prefix=[0, 3]),
                                  [[[0, 1], [0, 2], [0, 3], [0, 4]], [[0, 3], [0, 3], [0, 3], [0, 4]]])
    np.testing.assert_array_equal(gpu_op.attention_spans(4, documents=[5, 5, 5, 2]), [[0, 3], [0, 3], [0, 3], [3, 4]])
    with pytest.raises(ValueError):
        gpu_op.attention_spans(4, documents=[1, 2])


# ------------------------------------------------------------------------------- refusals

def _heads(parts, positions, frequencies, eps=1e-6, slots=None):
    _refused(gpu_op.head_rotary, parts, positions, frequencies, 1.0, False, eps, slots)


def test_head_rotary_refuses():
    part = gpu_op.head_part
    x, y, g, p, f = _Fake((6, 24)), _Fake((6, 24)), _Fake((8,)), _Fake((6,)), _Fake((4,))
    good = part(x, g, y, 3)
    _heads([], p, f)
    _heads([good] * 5, p, f)
    _heads([good], None, f)
    _heads([good], p, None)
    _heads([good], _Fake((4,)), f)                 # no divisor of the rows
    _heads([good], p, _Fake((5,)))                 # more pairs than a head has
    _heads([good], p, _Fake((2, 2)))
    _heads([good], p, f, eps=-1.0)
    _heads([good], p, f, eps=float("nan"))
    _heads([part(x, g, y, 5)], p, f)
    _heads([part(x, g, y, 0)], p, f)
    _heads([part(_Fake((1, 6, 4, 6)), g, _Fake((1, 6, 4, 6)), 3)], p, f)
    _heads([part(x, _Fake((7,)), y, 3)], p, f)
    _heads([part(x, g, _Fake((6, 16)), 3)], p, f)
    _heads([part(x, g, _Fake((6, 24), device=False), 3)], p, f)
    _heads([part(x, g, _Fake((6, 24), dev_id=1), 3)], p, f)
    _heads([good, part(_Fake((5, 24)), g, _Fake((5, 24)), 3)], p, f)
    _heads([good, part(_Fake((6, 16)), None, _Fake((6, 16)), 4)], p, f)   # heads of another length
    _heads([good, part(_Fake((6, 24)), g, y, 3)], p, f)                   # one output twice
    _heads([part(x, g, _Fake((6, 24), data=x.handle.contents.data + 4), 3)], p, f)
    _heads([part(x, g, y, 3), part(y, g, _Fake((6, 24)), 3)], p, f)       # what another part writes
    _heads([part(_Fake((1, 1026)), None, _Fake((1, 1026)), 1)], _Fake((1,)), f)
    cache, slots = _Fake((2, 9, 24)), _Fake((2, 3))
    placed = part(x, g, cache, 3, place=True)
    _heads([placed], p, f)
    _heads([placed], p, f, slots=_Fake((6,)))
    _heads([placed], p, f, slots=_Fake((2, 4)))
    _heads([part(x, g, _Fake((17, 24)), 3, place=True)], p, f, slots=slots)
    _heads([placed, part(_Fake((6, 24)), g, _Fake((2, 8, 24)), 3, place=True)], p, f, slots=slots)
    _heads([part(x, g, _Fake((2, 9, 24), data=x.handle.contents.data), 3, place=True)], p, f, slots=slots)


def test_head_rotary_backward_refuses():
    part = gpu_op.head_gradient_part
    x, dy, dx, g, dg, p, f = _Fake((6, 24)), _Fake((6, 24)), _Fake((6, 24)), _Fake((8,)), _Fake((8,)), _Fake((6,)), _Fake((4,))

    def refused(parts, positions=p, frequencies=f, eps=1e-6):
        _refused(gpu_op.head_rotary_backward, parts, positions, frequencies, 1.0, True, eps)
    refused([])
    refused([part(x, g, dy, None, None, 3)])
    refused([part(None, g, dy, dx, None, 3)])
    refused([part(x, None, dy, dx, dg, 3)])
    refused([part(_Fake((5, 24)), g, dy, dx, None, 3)])
    refused([part(x, g, dy, _Fake((6, 16)), None, 3)])
    refused([part(x, g, dy, dx, _Fake((7,)), 3)])
    refused([part(x, g, dy, x, None, 3)])
    refused([part(x, g, dy, dx, g, 3)])
    refused([part(x, g, dy, dx, dg, 3), part(_Fake((6, 24)), g, _Fake((6, 24)), _Fake((6, 24)), dg, 3)])
    refused([part(x, g, dy, _Fake((6, 24), data=dy.handle.contents.data + 4), None, 3)])
    refused([part(x, g, dy, dx, dg, 3)], positions=None)
    refused([part(x, g, dy, dx, dg, 3)], frequencies=_Fake((9,)))
    refused([part(x, g, dy, dx, dg, 3)], eps=-1.0)


def test_attention_refuses():
    q, k, v, o, s = _Fake((6, 32)), _Fake((8, 16)), _Fake((8, 16)), _Fake((6, 32)), _Fake((2, 4, 3))
    numbers = (2, 4, 2, 0.5, 0.0, False)

    def refused(q=q, k=k, v=v, spans=None, slopes=None, o=o, s=s, numbers=numbers):
        _refused(gpu_op.attention_forward, q, k, v, spans, slopes, o, s, *numbers)
    refused(o=None, s=None)
    refused(v=_Fake((8, 32)))
    refused(k=_Fake((8, 24)), v=_Fake((8, 24)))
    refused(q=_Fake((7, 32)), o=_Fake((7, 32)))
    refused(k=_Fake((7, 16)), v=_Fake((7, 16)))
    refused(o=_Fake((6, 16)))
    refused(s=_Fake((2, 4, 4)))
    refused(o=_Fake((6, 32), device=False))
    refused(o=_Fake((6, 32), dev_id=1))
    refused(o=_Fake((6, 32), data=q.handle.contents.data))
    refused(s=_Fake((2, 4, 3), data=o.handle.contents.data + 8))
    refused(spans=_Fake((2, 3)))
    refused(spans=_Fake((2, 2)))
    refused(spans=_Fake((3, 2), device=False))
    refused(slopes=_Fake((3,)))
    for bad in ((2, 4, 3, 0.5, 0.0, False), (2, 0, 0, 0.5, 0.0, False), (-1, 4, 2, 0.5, 0.0, False), (2, 4, 2, 0.0, 0.0, False),
                (2, 4, 2, -1.0, 0.0, False), (2, 4, 2, float("nan"), 0.0, False), (2, 4, 2, float("inf"), 0.0, False),
                (2, 4, 2, 0.5, -1.0, False), (2, 4, 2, 0.5, float("nan"), False), (2, 5, 1, 0.5, 0.0, False)):
        refused(numbers=bad)
    wide = _Fake((2, 257))
    refused(q=wide, k=_Fake((2, 257)), v=_Fake((2, 257)), o=_Fake((2, 257)), s=_Fake((2, 1, 1)), numbers=(2, 1, 1, 0.5, 0.0, False))
    long = (1 << 24) + 1
    refused(k=_Fake((2 * long, 16)), v=_Fake((2 * long, 16)))
    refused(q=_Fake((1 << 24, 64)), k=_Fake((1 << 24, 64)), v=_Fake((1 << 24, 64)), o=_Fake((1 << 24, 64)), s=None,
            numbers=(1 << 24, 64, 64, 0.5, 0.0, False))   # more heads than a launch has workgroups


def test_attention_backward_refuses():
    q, k, v, o, s, do = _Fake((6, 32)), _Fake((8, 16)), _Fake((8, 16)), _Fake((6, 32)), _Fake((2, 4, 3)), _Fake((6, 32))
    dq, dk, dv = _Fake((6, 32)), _Fake((8, 16)), _Fake((8, 16))

    def refused(o=o, s=s, do=do, dq=dq, dk=dk, dv=dv, numbers=(2, 4, 2, 0.5, 0.0, True)):
        _refused(gpu_op.attention_backward, q, k, v, None, None, o, s, do, dq, dk, dv, *numbers)
    refused(dq=None, dk=None, dv=None)
    refused(o=_Fake((6, 16)))
    refused(s=_Fake((2, 4)))
    refused(do=_Fake((6, 32), device=False))
    refused(dq=_Fake((8, 16)))
    refused(dk=_Fake((6, 32)))
    refused(dv=_Fake((8, 16), dev_id=1))
    refused(dk=dv)
    refused(dq=do)
    refused(dq=_Fake((6, 32), data=s.handle.contents.data))
    refused(dv=v)
    refused(numbers=(2, 4, 2, 0.5, -2.0, True))


def test_the_structures_are_those_of_the_header():
    assert ctypes.sizeof(gpu_op.HeadPart) == 40 and gpu_op.HeadPart.heads.offset == 24
    assert ctypes.sizeof(gpu_op.HeadGradientPart) == 48 and gpu_op.HeadGradientPart.heads.offset == 40


def test_spans_with_positions():
    np.testing.assert_array_equal(gpu_op.attention_spans(2, 9, causal=True, used=[4, 9], positions=True),
                                  [[[0, 3, 2], [0, 4, 3]], [[0, 8, 7], [0, 9, 8]]])
    np.testing.assert_array_equal(gpu_op.attention_spans(2, 3, positions=True), [[0, 3, 1], [0, 3, 2]])
    spans = gpu_op.attention_spans(3, documents=[[5, 5, 5], [1, 2, 2]], positions=True)
    np.testing.assert_array_equal(spans, [[[0, 3, 0], [0, 3, 1], [0, 3, 2]], [[0, 1, 0], [1, 3, 1], [1, 3, 2]]])
    assert spans.dtype == np.float32


def test_attention_refuses_spans_of_other_widths():
    q, k, v, o, s = _Fake((6, 32)), _Fake((8, 16)), _Fake((8, 16)), _Fake((6, 32)), _Fake((2, 4, 3))
    for shape in ((3, 4), (3, 1), (6,), (9,), (2, 2, 3), (3, 3, 3), (2, 3, 4)):
        _refused(gpu_op.attention_forward, q, k, v, _Fake(shape), None, o, s, 2, 4, 2, 0.5, 0.0, False)


def test_attention_refuses_numbers_at_the_ends_of_the_range():
    """A cap that is meant as none, one that leaves nothing, and scales whose product or quotient is no number with digits."""
    q, k, v, o, s = _Fake((6, 32)), _Fake((8, 16)), _Fake((8, 16)), _Fake((6, 32)), _Fake((2, 4, 3))
    grads = _Fake((6, 32)), _Fake((6, 32)), _Fake((8, 16)), _Fake((8, 16))
    largest = float(np.finfo(np.float32).max)
    for scale, cap in ((0.5, largest), (0.5, 1e-39), (1e-20, 1e20), (1e20, 1e-20), (largest, 0.0)):
        _refused(gpu_op.attention_forward, q, k, v, None, None, o, s, 2, 4, 2, scale, cap, False)
        _refused(gpu_op.attention_backward, q, k, v, None, None, o, s, *grads, 2, 4, 2, scale, cap, False)


def test_frequencies_refuse_parts_without_extent():
    for slow, fast in ((1.0, 1.0), (32.0, 1.0), (float("nan"), 32.0)):
        with pytest.raises(ValueError):
            gpu_op.rotary_frequencies(8, factor=4, context=2048, slow=slow, fast=fast)
