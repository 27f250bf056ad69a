"""The operators of a feed-forward sublayer together: as calls, as a training graph of each executor, and in a captured
graph."""
import ctypes
import random

import numpy as np
import pytest

import feed_forward_ref as ref

pytestmark = pytest.mark.gpu

EPS = 1e-5


def _values(rows, width, inner, seed):
    rng = np.random.RandomState(seed)

    def normal(*shape):
        return rng.normal(0, 1, shape)
    v = {"x": normal(rows, width) * 2 + 0.5, "gamma": 1 + 0.2 * normal(width), "beta": 0.1 * normal(width),
         "gate": normal(width, inner) / np.sqrt(width), "up": normal(width, inner) / np.sqrt(width),
         "down": normal(inner, width) / np.sqrt(inner), "dy": normal(rows, width)}
    return {k: a.astype(np.float32) for k, a in v.items()}


def _reference(v, mask):
    """Value and gradients of x + mask * (gated(norm(x)) down) in float64"""
    v = {k: a.astype(np.float64) for k, a in v.items()}
    norm = ref.Norm(v["x"], v["gamma"], v["beta"], EPS)
    g, u = norm.y @ v["gate"], norm.y @ v["up"]
    act, slope, _ = ref.act_and_slope(g, "silu")
    h = act * u
    out = {"y": v["x"] + mask * (h @ v["down"])}
    do = v["dy"] * mask
    dh = do @ v["down"].T
    dg, du = dh * u * slope, dh * act
    (dx, _), (dgamma, _), (dbeta, _) = norm.backward(dg @ v["gate"].T + du @ v["up"].T)
    out.update(dx=dx + v["dy"], dgamma=dgamma, dbeta=dbeta, dgate=norm.y.T @ dg, dup=norm.y.T @ du, ddown=h.T @ do)
    return out


def _near(got, value, what):
    """Sums of thousands of products, each operand a result itself: the errors add up as in a random walk, far below 1e-5 of the result's
    size (a wrong term is of that size)."""
    off = np.linalg.norm(got - value) / max(np.linalg.norm(value), 1e-30)
    assert off <= 1e-5, "%s is %.2g off" % (what, off)


@pytest.mark.parametrize("rows,width,inner", [(1, 48, 80), (7, 33, 65), (130, 128, 300), (300, 272, 520)])
def test_calls_in_a_row(rt, rows, width, inner):
    from tinyflow_amd import gpu_op, ndarray
    v = _values(rows, width, inner, rows)
    a = {k: ndarray.array(x, ctx=rt.ctx) for k, x in v.items()}

    def empty(*shape):
        return ndarray.empty(shape, ctx=rt.ctx)
    n, pre, h, o, y, do, dh, dn, dx = (empty(*s) for s in ((rows, width), (2, rows, inner), (rows, inner), (rows, width),
                                                           (rows, width), (rows, width), (rows, inner), (rows, width),
                                                           (rows, width)))
    d = {k: empty(*v[k].shape) for k in ("gamma", "beta", "gate", "up", "down")}
    p, seed, offset = 0.2, 77, 3
    gpu_op.layer_norm_forward(a["x"], a["gamma"], a["beta"], n, EPS, rt.stream)
    assert gpu_op.gated_feed_forward(n, a["gate"], a["up"], pre, h, "silu", rt.stream) == 0
    gpu_op.matrix_multiply(h, False, a["down"], False, o, rt.cublas, rt.stream)
    gpu_op.counter_dropout(o, a["x"], y, p, seed, offset, rt.stream)
    gpu_op.counter_dropout(a["dy"], None, do, p, seed, offset, rt.stream)
    gpu_op.matrix_multiply(h, True, do, False, d["down"], rt.cublas, rt.stream)
    gpu_op.matrix_multiply(do, False, a["down"], True, dh, rt.cublas, rt.stream)
    assert gpu_op.gated_feed_forward_backward(n, a["gate"], a["up"], pre, dh, dn, d["gate"], d["up"], "silu", rt.stream) == 0
    assert gpu_op.layer_norm_backward(a["x"], a["gamma"], dn, dx, d["gamma"], d["beta"], EPS, rt.stream) == 0
    gpu_op.matrix_elementwise_add(dx, a["dy"], dx, rt.stream)
    mask = ref.kept(rows * width, p, seed, offset).reshape(rows, width) / (1 - float(np.float32(p)))
    wanted = _reference(v, mask)
    got = dict(y=y, dx=dx, **{"d" + k: arr for k, arr in d.items()})
    for name, value in wanted.items():
        _near(got[name].asnumpy(), value, name)


# ----------------------------------------------------------------------------- as a graph

ROWS, WIDTH, INNER, CLASSES = 70, 40, 72, 6


def _graph(dropout):
    from tinyflow_amd import autodiff as ad
    X, y_ = ad.Placeholder("X"), ad.Placeholder("y_")
    rng = np.random.RandomState(5)
    variables = {}

    def variable(name, value):
        node = ad.Variable(name)
        variables[node] = np.asarray(value, np.float32)
        return node
    x = ad.matmul_op(X, variable("embed", rng.normal(0, 0.5, (12, WIDTH))))
    for layer in range(2):
        n = ad.layer_norm_forward_op(x, variable("gamma%d" % layer, 1 + 0.1 * rng.normal(0, 1, WIDTH)),
                                     variable("beta%d" % layer, 0.1 * rng.normal(0, 1, WIDTH)), EPS)
        h = ad.gated_feed_forward(n, variable("gate%d" % layer, rng.normal(0, 0.2, (WIDTH, INNER))),
                                  variable("up%d" % layer, rng.normal(0, 0.2, (WIDTH, INNER))), ("silu", "gelu")[layer])
        o = ad.matmul_op(h, variable("down%d" % layer, rng.normal(0, 0.2, (INNER, WIDTH))))
        x = ad.counter_dropout_op(o, dropout, residual=x, seed=100 + layer)
    loss = ad.softmaxcrossentropy_op(ad.matmul_op(x, variable("head", rng.normal(0, 0.2, (WIDTH, CLASSES)))), y_)
    data = rng.normal(0, 1, (ROWS, 12)).astype(np.float32)
    labels = np.eye(CLASSES, dtype=np.float32)[rng.randint(0, CLASSES, ROWS)]
    return loss, X, y_, variables, data, labels


def _step_in_float64(values, data, labels, dropout, offset):
    """Loss and gradients of _graph, by name; the loss's gradient is not divided by the batch (softmaxcrossentropy_op)."""
    v = {k: a.astype(np.float64) for k, a in values.items()}
    x, kept = data.astype(np.float64) @ v["embed"], []
    for layer in range(2):
        norm = ref.Norm(x, v["gamma%d" % layer], v["beta%d" % layer], EPS)
        g, u = norm.y @ v["gate%d" % layer], norm.y @ v["up%d" % layer]
        act, slope, _ = ref.act_and_slope(g, ("silu", "gelu")[layer])
        mask = ref.kept(x.size, dropout, 100 + layer, offset).reshape(x.shape) / (1 - float(np.float32(dropout)))
        kept.append((norm, g, u, act, slope, mask))
        x = x + mask * ((act * u) @ v["down%d" % layer])
    logits = x @ v["head"]
    p = np.exp(logits - logits.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    loss = -(labels * np.log(p)).sum() / len(data)
    grads = {"head": x.T @ (p - labels)}
    dx = (p - labels) @ v["head"].T
    for layer in (1, 0):
        norm, g, u, act, slope, mask = kept[layer]
        do = dx * mask
        grads["down%d" % layer] = (act * u).T @ do
        dh = do @ v["down%d" % layer].T
        dg, du = dh * u * slope, dh * act
        grads["gate%d" % layer], grads["up%d" % layer] = norm.y.T @ dg, norm.y.T @ du
        (dn, _), (grads["gamma%d" % layer], _), (grads["beta%d" % layer], _) = norm.backward(
            dg @ v["gate%d" % layer].T + du @ v["up%d" % layer].T)
        dx = dx + dn
    grads["embed"] = data.astype(np.float64).T @ dx
    return loss, grads


@pytest.mark.parametrize("dropout", [0.0, 0.3])
def test_training_steps(rt, dropout):
    """Two steps: every gradient of each, with the masks of its own evaluation."""
    from tinyflow_amd.TrainExecute import TrainExecutor
    loss, X, y_, variables, data, labels = _graph(dropout)
    rate = 1e-3
    ex = TrainExecutor(loss, rate)
    ex.init_Variable(dict(variables))
    values = {n.name: v for n, v in variables.items()}
    for step in range(2):
        out = ex.run({X: data, y_: labels})
        wanted, grads = _step_in_float64(values, data, labels, dropout, step)
        assert abs(out[0].asnumpy()[0] - wanted) <= 1e-5 * abs(wanted)
        for node, g in zip(ex.Variable_node_list, ex.Variable_node_grad_list):
            _near(ex.value_of(g).asnumpy(), grads[node.name], "gradient of %s, step %d" % (node.name, step))
        values = {n.name: ex.value_of(n).asnumpy() for n in variables}
    ex.close()


def test_executors_agree_to_the_bit(rt):
    """One call for several nodes, a call for each, and the swap executor's released and recomputed values."""
    from tinyflow_amd import TrainExecute
    from tinyflow_amd.SwapExecute import SwapExecutor
    results = []
    for kind in ("joined", "apart", "swap", "recompute"):
        loss, X, y_, variables, data, labels = _graph(0.25)
        if kind in ("joined", "apart"):
            find = TrainExecute.find_siblings
            if kind == "apart":
                TrainExecute.find_siblings = lambda order, unavailable: {}
            try:
                ex = TrainExecute.TrainExecutor(loss, 1e-2)
                ex.init_Variable(dict(variables))
                runs = [ex.run({X: data, y_: labels}) for _ in range(3)]
            finally:
                TrainExecute.find_siblings = find
        else:
            ex = SwapExecutor(loss, 1e-2, swap=True, min_swap_bytes=1, recompute=kind == "recompute")
            ex.init_Variable(dict(variables))
            runs = [ex.run({X: data, y_: labels}) for _ in range(3)]
            if kind == "recompute":
                assert ex.swap_report()["recomputed"] > 0
        results.append([a.asnumpy() for a in runs[-1]])
        if hasattr(ex, "close"):
            ex.close()
    for other in results[1:]:
        assert len(other) == len(results[0])
        for a, b in zip(results[0], other):
            np.testing.assert_array_equal(a, b)


def test_adam(rt):
    from tinyflow_amd.TrainExecuteAdam import TrainExecutor
    loss, X, y_, variables, data, labels = _graph(0.1)
    ex = TrainExecutor(loss, 1e-3)
    ex.init_Variable(dict(variables))
    ex.run({X: data, y_: labels})
    _, grads = _step_in_float64({n.name: v for n, v in variables.items()}, data, labels, 0.1, 0)
    for node, g in zip(ex.Variable_node_list, ex.Variable_node_grad_list):
        _near(ex.value_of(g).asnumpy(), grads[node.name], "gradient of %s" % node.name)
    ex.close()


def test_a_seed_from_pythons_generator(rt):
    """The same state of ``random``, the same masks."""
    from tinyflow_amd import autodiff as ad
    from tinyflow_amd.TrainExecute import TrainExecutor
    outs = []
    for state in (1, 1, 2):
        random.seed(state)
        w = ad.Variable("w")
        loss = ad.reduce_sum_op(ad.counter_dropout_op(w, 0.5))
        ex = TrainExecutor(loss, 0.0)
        ex.init_Variable({w: np.ones((40, 50), np.float32)})
        ex.run({})
        first = ex.value_of(ex.Variable_node_grad_list[0]).asnumpy()
        ex.run({})
        outs.append((first, ex.value_of(ex.Variable_node_grad_list[0]).asnumpy()))
        ex.close()
    for a, b in zip(outs[0], outs[1]):
        np.testing.assert_array_equal(a, b)
    assert (outs[0][0] != outs[0][1]).any() and (outs[0][0] != outs[2][0]).any()


# ------------------------------------------------------------------------ captured graphs

def test_calls_without_scratch_in_a_captured_graph(rt):
    import torch
    from tinyflow_amd import gpu_op, ndarray
    stream = gpu_op.create_cudaStream()
    v = _values(3, 64, 96, 2)
    a = {k: ndarray.array(x, ctx=rt.ctx) for k, x in v.items()}
    n, h, y = (ndarray.array(np.zeros(s, np.float32), ctx=rt.ctx) for s in ((3, 64), (3, 96), (3, 64)))
    dx, dgamma, dpre = (ndarray.empty(s, ctx=rt.ctx) for s in ((3, 64), (64,), (2, 3, 96)))

    def calls():
        gpu_op.layer_norm_forward(a["x"], a["gamma"], a["beta"], n, EPS, stream)
        assert gpu_op.gated_feed_forward(n, a["gate"], a["up"], None, h, "silu", stream) == 0
        gpu_op.counter_dropout(n, a["x"], y, 0.5, 9, 4, stream)
        assert gpu_op.layer_norm_backward(a["x"], a["gamma"], n, dx, None, None, EPS, stream) == 0
    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    external = torch.cuda.ExternalStream(ctypes.cast(stream.contents, ctypes.c_void_p).value)
    with torch.cuda.graph(graph, stream=external):
        calls()
        # what takes scratch says so, and leaves the capture as it is
        with pytest.raises(RuntimeError):
            gpu_op.layer_norm_backward(a["x"], a["gamma"], n, dx, dgamma, None, EPS, stream)
        with pytest.raises(RuntimeError):
            gpu_op.gated_feed_forward_backward(n, a["gate"], a["up"], None, dpre, dx, None, None, "silu", stream)
    for replay in range(3):
        x = _values(3, 64, 96, 10 + replay)["x"]
        a["x"][:] = x
        graph.replay()
        torch.cuda.synchronize()
        got = [arr.asnumpy() for arr in (n, h, y, dx)]
        for arr in (n, h, y, dx):
            gpu_op.array_set(arr, 3.0, rt.stream)
        calls()
        for g, arr in zip(got, (n, h, y, dx)):
            np.testing.assert_array_equal(g, arr.asnumpy())
    gpu_op.destroy_cudaStream(stream)


# ------------------------------------------------------------------------ calls at once

def test_two_threads_with_a_stream_each(rt):
    """Scratch, tickets and the pool under calls that two threads make at the same time: the same bits as one after the other."""
    import threading
    from tinyflow_amd import gpu_op, ndarray
    shapes = [(24, 300, 520), (700, 520, 1000)]   # folded in one launch; on pairs, with planes and pieces
    work = []
    for t, (rows, width, inner) in enumerate(shapes):
        v = _values(rows, width, inner, 40 + t)
        a = {k: ndarray.array(x, ctx=rt.ctx) for k, x in v.items()}
        outs = [ndarray.empty(s, ctx=rt.ctx) for s in ((rows, width), (2, rows, inner), (rows, inner), (rows, width), (width, inner),
                                                       (width, inner), (rows, width), (width,), (width,))]
        work.append((a, outs, gpu_op.create_cudaStream()))

    def calls(a, outs, stream):
        n, pre, h, dx, dgate, dup, dn, dgamma, dbeta = outs
        gpu_op.layer_norm_forward(a["x"], a["gamma"], a["beta"], n, EPS, stream)
        assert gpu_op.gated_feed_forward(n, a["gate"], a["up"], pre, h, "silu", stream) == 0
        assert gpu_op.gated_feed_forward_backward(n, a["gate"], a["up"], pre, h, dx, dgate, dup, "silu", stream) == 0
        assert gpu_op.layer_norm_backward(a["x"], a["gamma"], dx, dn, dgamma, dbeta, EPS, stream) == 0

    wanted = []
    for w in work:
        calls(*w)
        wanted.append([o.asnumpy() for o in w[1]])
    failures = []

    def run(w):
        try:
            for _ in range(30):
                calls(*w)
        except Exception as e:   # the test's thread reports it
            failures.append(e)
    threads = [threading.Thread(target=run, args=(w,)) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    for w, values in zip(work, wanted):
        for o, value in zip(w[1], values):
            np.testing.assert_array_equal(o.asnumpy(), value)
        gpu_op.destroy_cudaStream(w[2])
