"""The operators of an attention sublayer together: as calls, token by token over a cache, as a training graph of each executor, in a captured graph
and from two threads."""
import ctypes
import threading

import numpy as np
import pytest

import attention_ref as ref
import feed_forward_ref as ff

pytestmark = pytest.mark.gpu

EPS, HEAD_EPS = 1e-5, 1e-6


def _normal(rng, *shape):
    return rng.normal(0, 1, shape).astype(np.float32)


def _weights(rng, width, h, hk, d):
    w = {"gamma": 1 + 0.2 * _normal(rng, width), "beta": 0.1 * _normal(rng, width), "wq": _normal(rng, width, h * d) / np.sqrt(width),
         "wk": _normal(rng, width, hk * d) / np.sqrt(width), "wv": _normal(rng, width, hk * d) / np.sqrt(width),
         "wo": _normal(rng, h * d, width) / np.sqrt(h * d), "gq": 1 + 0.2 * _normal(rng, d), "gk": 1 + 0.2 * _normal(rng, d)}
    return {k: v.astype(np.float32) for k, v in w.items()}


class _Sublayer(object):
    """x + attention(rotated(n wq), rotated(n wk), n wv) wo with n = norm(x), and its gradients, in float64"""

    def __init__(self, v, x, b, h, hk, d, frequencies, spans, causal):
        v = {k: a.astype(np.float64) for k, a in v.items()}
        self.v, self.x, self.sizes = v, x.astype(np.float64), (b, h, hk, d)
        self.norm = ff.Norm(self.x, v["gamma"], v["beta"], EPS)
        n, rows = self.norm.y, len(x)
        positions = np.arange(rows // b)
        self.q = ref.Heads((n @ v["wq"]).reshape(rows, h, d), v["gq"], positions, frequencies, 1.0, False, HEAD_EPS)
        self.k = ref.Heads((n @ v["wk"]).reshape(rows, hk, d), v["gk"], positions, frequencies, 1.0, False, HEAD_EPS)
        self.att = ref.Attention(self.q.y.reshape(b, -1, h, d), self.k.y.reshape(b, -1, hk, d), (n @ v["wv"]).reshape(b, -1, hk, d), spans, None,
                                 d ** -0.5, 0.0, causal)
        self.y = self.x + self.att.out.reshape(rows, -1) @ v["wo"]

    def backward(self, dy):
        v, n, rows = self.v, self.norm.y, len(self.x)
        b, h, hk, d = self.sizes
        out = self.att.out.reshape(rows, -1)
        inner = self.att.backward(self.att.out, self.att.stat, (dy @ v["wo"].T).reshape(b, -1, h, d))
        (dq, _), (dgq, _) = self.q.backward(inner[0][0].reshape(rows, h, d))
        (dk, _), (dgk, _) = self.k.backward(inner[1][0].reshape(rows, hk, d))
        dq, dk, dv = dq.reshape(rows, -1), dk.reshape(rows, -1), inner[2][0].reshape(rows, -1)
        (dx, _), (dgamma, _), (dbeta, _) = self.norm.backward(dq @ v["wq"].T + dk @ v["wk"].T + dv @ v["wv"].T)
        return dict(x=dx + dy, gamma=dgamma, beta=dbeta, wq=n.T @ dq, wk=n.T @ dk, wv=n.T @ dv, wo=out.T @ dy, gq=dgq, gk=dgk)


def _near(got, value, what):
    """Sums of thousands of products, each operand a result itself: the errors add up as in a random walk, far below 2e-5 of the result's
    size (a wrong term is of that size)."""
    off = np.linalg.norm(got - value) / max(np.linalg.norm(value), 1e-30)
    assert off <= 2e-5, "%s is %.2g off" % (what, off)


@pytest.mark.parametrize("b,t,width,h,hk,d,spans", [(1, 1, 24, 2, 1, 16, False), (2, 9, 40, 4, 2, 12, True), (2, 70, 64, 6, 3, 32, False),
                                                    (1, 300, 128, 4, 4, 64, True)])
def test_calls_in_a_row(rt, b, t, width, h, hk, d, spans):
    from tinyflow_amd import gpu_op, ndarray
    rng = np.random.RandomState(t)
    v, x, dy = _weights(rng, width, h, hk, d), _normal(rng, b * t, width) * 2, _normal(rng, b * t, width)
    f = gpu_op.rotary_frequencies(d)
    mask = gpu_op.attention_spans(t, causal=True, prefix=[t // 3] * b) if spans else None
    want = _Sublayer(v, x, b, h, hk, d, f, mask, not spans)
    a = {k: ndarray.array(val, ctx=rt.ctx) for k, val in v.items()}
    ax, ady, af, ap = (ndarray.array(val, ctx=rt.ctx) for val in (x, dy, f, np.arange(t, dtype=np.float32)))
    am = None if mask is None else ndarray.array(mask, ctx=rt.ctx)

    def empty(*shape):
        return ndarray.empty(shape, ctx=rt.ctx)
    rows = b * t
    n, y, p, dn, dn2 = (empty(rows, width) for _ in range(5))
    q, qr, att, datt, dq, dqr = (empty(rows, h * d) for _ in range(6))
    k, kr, vv, dk, dkr, dv = (empty(rows, hk * d) for _ in range(6))
    stat = empty(b, h, t)
    g = {name: empty(*v[name].shape) for name in v}

    def multiply(x, tx, y, ty, out):
        gpu_op.matrix_multiply(x, tx, y, ty, out, rt.cublas, rt.stream)
    gpu_op.layer_norm_forward(ax, a["gamma"], a["beta"], n, EPS, rt.stream)
    for w, out in (("wq", q), ("wk", k), ("wv", vv)):
        multiply(n, False, a[w], False, out)
    gpu_op.head_rotary([gpu_op.head_part(q, a["gq"], qr, h), gpu_op.head_part(k, a["gk"], kr, hk)], ap, af, 1.0, False, HEAD_EPS, None, rt.stream)
    numbers = (b, h, hk, d ** -0.5, 0.0, not spans, rt.stream)
    assert gpu_op.attention_forward(qr, kr, vv, am, None, att, stat, *numbers) == 0
    multiply(att, False, a["wo"], False, p)
    gpu_op.matrix_elementwise_add(p, ax, y, rt.stream)
    multiply(att, True, ady, False, g["wo"])
    multiply(ady, False, a["wo"], True, datt)
    assert gpu_op.attention_backward(qr, kr, vv, am, None, att, stat, datt, dqr, dkr, dv, *numbers) == 0
    part = gpu_op.head_gradient_part
    assert gpu_op.head_rotary_backward([part(q, a["gq"], dqr, dq, g["gq"], h), part(k, a["gk"], dkr, dk, g["gk"], hk)], ap, af, 1.0, False,
                                       HEAD_EPS, rt.stream) == 0
    for w, dz, out in (("wq", dq, dn), ("wk", dk, p), ("wv", dv, dn2)):
        multiply(n, True, dz, False, g[w])
        multiply(dz, False, a[w], True, out)
    gpu_op.matrix_elementwise_add(dn, p, dn, rt.stream)
    gpu_op.matrix_elementwise_add(dn, dn2, dn, rt.stream)
    assert gpu_op.layer_norm_backward(ax, a["gamma"], dn, p, g["gamma"], g["beta"], EPS, rt.stream) == 0
    gpu_op.matrix_elementwise_add(p, ady, dn, rt.stream)
    _near(y.asnumpy(), want.y, "y")
    if t == 1:
        return   # one token attends to itself alone: the gradients of queries and keys are nothing but rounding
    for name, value in want.backward(dy.astype(np.float64)).items():
        _near((dn if name == "x" else g[name]).asnumpy(), value, "d" + name)


@pytest.mark.parametrize("h,hk,d", [(4, 1, 32), (6, 3, 80)])
def test_token_by_token_is_the_whole_sequence(rt, h, hk, d):
    """A prompt at once, then tokens one by one: each row placed in the cache and read back by the next ones."""
    from tinyflow_amd import gpu_op, ndarray
    rng = np.random.RandomState(d)
    b, prompt, more, capacity = 2, 37, 6, 64
    t = prompt + more
    q, k, v = (_normal(rng, b, t, n, d) for n in (h, hk, hk))
    gq, gk, f = 1 + 0.1 * _normal(rng, d), 1 + 0.1 * _normal(rng, d), gpu_op.rotary_frequencies(d)
    rotated = [ref.Heads(x.reshape(b * t, -1, d), g, np.arange(t), f, 1.0, True, HEAD_EPS).y.reshape(x.shape) for x, g in ((q, gq), (k, gk))]
    want = ref.Attention(*rotated, v, None, None, d ** -0.5, 0.0, True)

    def device(x):
        return ndarray.array(np.ascontiguousarray(x, np.float32), ctx=rt.ctx)
    agq, agk, af = device(gq), device(gk), device(f)
    k_cache, v_cache = (device(np.full((b, capacity, hk * d), np.nan)) for _ in range(2))   # what is not written is never read
    start = 0
    for n in [prompt] + [1] * more:
        new = slice(start, start + n)
        aq, ak, av = (device(x[:, new].reshape(b, n, -1)) for x in (q, k, v))
        qr, out = device(np.zeros((b, n, h * d))), device(np.zeros((b, n, h * d)))
        positions, slots = device(np.arange(start, start + n)), device(np.tile(np.arange(start, start + n), (b, 1)))
        gpu_op.head_rotary([gpu_op.head_part(aq, agq, qr, h), gpu_op.head_part(ak, agk, k_cache, hk, place=True),
                            gpu_op.head_part(av, None, v_cache, hk, rotate=False, place=True)], positions, af, 1.0, True, HEAD_EPS, slots, rt.stream)
        start += n
        spans = device(gpu_op.attention_spans(n, capacity, causal=True, used=[start] * b))
        assert gpu_op.attention_forward(qr, k_cache, v_cache, spans, None, out, None, b, h, hk, d ** -0.5, 0.0, False, rt.stream) == 0
        _near(out.asnumpy().reshape(b, n, h, d), want.out[:, new], "tokens %d.." % (start - n))


def test_far_rows_of_a_long_cache(rt):
    """Rows whose offsets pass 2^31 elements: placed there and read from there."""
    from tinyflow_amd import gpu_op, ndarray
    rng = np.random.RandomState(3)
    h, hk, d, capacity, n = 4, 2, 128, (1 << 23) + 40, 21
    q, k, v = _normal(rng, 1, 1, h, d), _normal(rng, 1, n, hk, d), _normal(rng, 1, n, hk, d)
    ak, av, aq = (ndarray.array(x.reshape(1, x.shape[1], -1), ctx=rt.ctx) for x in (k, v, q))
    caches = [ndarray.empty((1, capacity, hk * d), ctx=rt.ctx) for _ in range(2)]
    for c in caches:
        gpu_op.array_set(c, 7.0, rt.stream)
    slots = ndarray.array((capacity - n + np.arange(n, dtype=np.float32))[None], ctx=rt.ctx)
    gpu_op.head_rotary([gpu_op.head_part(x, None, c, hk, rotate=False, place=True) for x, c in ((ak, caches[0]), (av, caches[1]))], None, None, 1.0,
                       False, HEAD_EPS, slots, rt.stream)
    out = ndarray.empty((1, 1, h * d), ctx=rt.ctx)
    spans = ndarray.array(np.array([[capacity - n, capacity]], np.float32), ctx=rt.ctx)
    want = ref.Attention(q, k, v, None, None, d ** -0.5)
    assert gpu_op.attention_forward(aq, *caches, spans, None, out, None, 1, h, hk, d ** -0.5, 0.0, False, rt.stream) == 0
    ref.assert_within(out.asnumpy().reshape(want.out.shape), want.out, want.out_tol, "out")


# ----------------------------------------------------------------------------- as a graph

B, T, WIDTH, HEADS, KEY_HEADS, DIM, CLASSES = 2, 24, 20, 4, 2, 12, 5


def _graph(masks):
    from tinyflow_amd import autodiff as ad, gpu_op
    rng = np.random.RandomState(5)
    X, y_ = ad.Placeholder("X"), ad.Placeholder("y_")
    feed = {"positions": np.arange(T, dtype=np.float32), "frequencies": gpu_op.rotary_frequencies(DIM)}
    if masks:
        feed["spans"] = gpu_op.attention_spans(T, causal=True, documents=np.repeat([0, 1, 2], T // 3)[None].repeat(B, 0))
    places = {name: ad.Placeholder(name) for name in feed}
    variables = {}

    def variable(name, value):
        node = ad.Variable(name)
        variables[node] = np.asarray(value, np.float32)
        return node
    x = ad.matmul_op(X, variable("embed", _normal(rng, 12, WIDTH)))
    for layer in range(2):
        w = {k: variable("%s%d" % (k, layer), val) for k, val in _weights(rng, WIDTH, HEADS, KEY_HEADS, DIM).items()}
        n = ad.layer_norm_forward_op(x, w["gamma"], w["beta"], EPS)
        x = x + ad.self_attention(n, w["wq"], w["wk"], w["wv"], w["wo"], B, HEADS, KEY_HEADS, (w["gq"], w["gk"]), places["positions"],
                                  places["frequencies"], spans=places.get("spans"), causal=not masks)
    loss = ad.softmaxcrossentropy_op(ad.matmul_op(x, variable("head", 0.2 * _normal(rng, WIDTH, CLASSES))), y_)
    feed = {places[name]: value for name, value in feed.items()}
    feed[X] = _normal(rng, B * T, 12)
    feed[y_] = np.eye(CLASSES, dtype=np.float32)[rng.randint(0, CLASSES, B * T)]
    return loss, X, y_, places, variables, feed


def _step_in_float64(values, feed, X, y_, places):
    """Loss and gradients of _graph, by name; the loss's gradient is not divided by the batch (softmaxcrossentropy_op)."""
    spans = feed.get(places.get("spans"))
    x, layers = feed[X].astype(np.float64) @ values["embed"].astype(np.float64), []
    for layer in range(2):
        v = {k[:-1]: a for k, a in values.items() if k.endswith(str(layer))}
        layers.append(_Sublayer(v, x, B, HEADS, KEY_HEADS, DIM, feed[places["frequencies"]], spans, spans is None))
        x = layers[-1].y
    logits = x @ values["head"].astype(np.float64)
    p = np.exp(logits - logits.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    labels = feed[y_]
    grads = {"head": x.T @ (p - labels)}
    dx = (p - labels) @ values["head"].astype(np.float64).T
    for layer in (1, 0):
        found = layers[layer].backward(dx)
        dx = found.pop("x")
        grads.update({"%s%d" % (k, layer): g for k, g in found.items()})
    grads["embed"] = feed[X].astype(np.float64).T @ dx
    return -(labels * np.log(p)).sum() / len(labels), grads


@pytest.mark.parametrize("masks", [False, True])
def test_training_steps(rt, masks):
    from tinyflow_amd.TrainExecute import TrainExecutor
    loss, X, y_, places, variables, feed = _graph(masks)
    ex = TrainExecutor(loss, 1e-3)
    ex.init_Variable(dict(variables))
    values = {n.name: v for n, v in variables.items()}
    for step in range(2):
        out = ex.run(feed)
        wanted, grads = _step_in_float64(values, feed, X, y_, places)
        assert abs(out[0].asnumpy()[0] - wanted) <= 1e-5 * abs(wanted)
        for node, g in zip(ex.Variable_node_list, ex.Variable_node_grad_list):
            _near(ex.value_of(g).asnumpy(), grads[node.name], "gradient of %s, step %d" % (node.name, step))
        values = {n.name: ex.value_of(n).asnumpy() for n in variables}
    ex.close()


def test_adam(rt):
    from tinyflow_amd.TrainExecuteAdam import TrainExecutor
    loss, X, y_, places, variables, feed = _graph(True)
    ex = TrainExecutor(loss, 1e-3)
    ex.init_Variable(dict(variables))
    ex.run(feed)
    _, grads = _step_in_float64({n.name: v for n, v in variables.items()}, feed, X, y_, places)
    for node, g in zip(ex.Variable_node_list, ex.Variable_node_grad_list):
        _near(ex.value_of(g).asnumpy(), grads[node.name], "gradient of %s" % node.name)
    ex.close()


def test_executors_agree_to_the_bit(rt):
    """One call for several nodes, a call for each, and the swap executor's released and recomputed values."""
    from tinyflow_amd import TrainExecute
    from tinyflow_amd.SwapExecute import SwapExecutor
    results = []
    for kind in ("joined", "apart", "swap", "recompute"):
        loss, _, _, _, variables, feed = _graph(True)
        if kind in ("joined", "apart"):
            find = TrainExecute.find_siblings
            if kind == "apart":
                TrainExecute.find_siblings = lambda order, unavailable: {}
            try:
                ex = TrainExecute.TrainExecutor(loss, 1e-2)
                ex.init_Variable(dict(variables))
                runs = [ex.run(feed) for _ in range(3)]
            finally:
                TrainExecute.find_siblings = find
        else:
            ex = SwapExecutor(loss, 1e-2, swap=True, min_swap_bytes=1, recompute=kind == "recompute")
            ex.init_Variable(dict(variables))
            runs = [ex.run(feed) for _ in range(3)]
        results.append([a.asnumpy() for a in runs[-1]])
        if hasattr(ex, "close"):
            ex.close()
    for other in results[1:]:
        assert len(other) == len(results[0])
        for a, b in zip(results[0], other):
            np.testing.assert_array_equal(a, b)


# ------------------------------------------------------------------------ captured graphs

def test_a_token_in_a_captured_graph(rt, monkeypatch):
    """Norm, rotation, placement and attention over a short cache take no scratch: replays have the bits of the eager calls.  What takes
    some says so, and leaves the capture as it is."""
    import torch
    from tinyflow_amd import gpu_op, ndarray
    stream = gpu_op.create_cudaStream()
    rng = np.random.RandomState(8)
    h, hk, d, capacity = 4, 2, 32, 50

    def device(x):
        return ndarray.array(np.ascontiguousarray(x, np.float32), ctx=rt.ctx)
    q, k, v = device(_normal(rng, 1, h * d)), device(_normal(rng, 1, hk * d)), device(_normal(rng, 1, hk * d))
    gamma, f, positions, slots = device(np.ones(d)), device(gpu_op.rotary_frequencies(d)), device([3]), device([[3]])
    spans, caches = device([[0, 4]]), [device(_normal(rng, 1, capacity, hk * d)) for _ in range(2)]
    qr, out, stat = device(np.zeros((1, h * d))), device(np.zeros((1, h * d))), device(np.zeros((1, h, 1)))
    numbers = (1, h, hk, d ** -0.5, 20.0, False, stream)
    long_k, big = device(_normal(rng, 4000, hk * d)), device(_normal(rng, 300, h * d))
    big_k, big_out, big_stat = device(_normal(rng, 300, hk * d)), device(np.zeros((300, h * d))), device(np.zeros((1, h, 300)))

    def calls():
        gpu_op.head_rotary([gpu_op.head_part(q, gamma, qr, h), gpu_op.head_part(k, gamma, caches[0], hk, place=True),
                            gpu_op.head_part(v, None, caches[1], hk, rotate=False, place=True)], positions, f, 1.0, False, HEAD_EPS, slots, stream)
        assert gpu_op.attention_forward(qr, *caches, spans, None, out, stat, *numbers) == 0
    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(ctypes.cast(stream.contents, ctypes.c_void_p).value)):
        calls()
        with pytest.raises(RuntimeError):
            gpu_op.attention_forward(qr, long_k, long_k, None, None, out, None, *numbers)
        with pytest.raises(RuntimeError):
            gpu_op.attention_forward(big, big_k, big_k, None, None, big_out, None, *numbers)
        with pytest.raises(RuntimeError):
            gpu_op.attention_backward(big, big_k, big_k, None, None, big_out, big_stat, big, big_out, None, None, *numbers)
    for replay in range(4):
        at = 4 + replay
        q[:], k[:], v[:] = _normal(rng, 1, h * d), _normal(rng, 1, hk * d), _normal(rng, 1, hk * d)
        positions[:], slots[:], spans[:] = np.float32([at]), np.float32([[at]]), np.float32([[0, at + 1]])
        graph.replay()
        torch.cuda.synchronize()
        arrays = [qr, out, stat] + caches
        got = [a.asnumpy() for a in arrays]
        for a in (qr, out, stat):
            gpu_op.array_set(a, 3.0, rt.stream)
        calls()
        for g, a in zip(got, arrays):
            np.testing.assert_array_equal(g, a.asnumpy())
    gpu_op.destroy_cudaStream(stream)


# ------------------------------------------------------------------------ calls at once

def test_two_threads_with_a_stream_each(rt):
    """Scratch and the pool under calls that two threads make at the same time: the same bits as one after the other."""
    from tinyflow_amd import gpu_op, ndarray
    work = []
    for seed, (b, tq, tk, h, hk, d) in enumerate([(2, 3, 900, 6, 2, 40), (1, 300, 300, 4, 2, 64)]):   # cut along the keys; on pairs
        rng = np.random.RandomState(seed)
        a = [ndarray.array(_normal(rng, *s), ctx=rt.ctx) for s in ((b, tq, h, d), (b, tk, hk, d), (b, tk, hk, d), (b, tq, h, d))]
        outs = [ndarray.empty(s, ctx=rt.ctx) for s in ((b, tq, h, d), (b, h, tq), (b, tq, h, d), (b, tk, hk, d), (b, tk, hk, d))]
        work.append((a, outs, (b, h, hk, d ** -0.5, 0.0, True), gpu_op.create_cudaStream()))

    def calls(a, outs, numbers, stream):
        assert gpu_op.attention_forward(*a[:3], None, None, *outs[:2], *numbers, stream) == 0
        assert gpu_op.attention_backward(*a[:3], None, None, *outs[:2], a[3], *outs[2:], *numbers, stream) == 0
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
        gpu_op.destroy_cudaStream(w[3])
