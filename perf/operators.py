"""The operators of a pre-norm feed-forward sublayer, y = x + dropout(gated(layer_norm(x)) W), as cases that can be
timed: layer norm, the gated feed-forward product and counter-based dropout, each forward and backward, and a run of
them together.

``own`` false: the operators in plain torch, fp32. ``own`` true: the calls that a user makes of ``tinyflow_amd.gpu_op``.
Everything is fp32, the one type of the package's arrays.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5


# ------------------------------------------------------------------------------ the cases

def _norm(name, direction, rows, cols):
    return {"name": name, "kind": "norm", "direction": direction, "rows": rows, "cols": cols}


def _drop(name, direction, count, dropout, offset):
    """``forward`` adds a residual, ``backward`` is the same mask on a gradient."""
    return {"name": name, "kind": "drop", "direction": direction, "count": count, "dropout": dropout, "offset": offset}


def _gated(name, direction, rows, width, inner, activation):
    """``serve``: the product alone; ``train``: with the projections that the backward pass reads; ``backward``."""
    return {"name": name, "kind": "gated", "direction": direction, "rows": rows, "width": width, "inner": inner,
            "activation": activation}


def _sublayer(name, rows, width, inner, dropout):
    return {"name": name, "kind": "sublayer", "rows": rows, "width": width, "inner": inner, "dropout": dropout}


def listed():
    return [
        # one token being generated: nothing but latency
        _norm("norm 1 token", "forward", 1, 1024),
        # the tokens of a training batch, a wide network
        _norm("norm 8192x2048", "forward", 8192, 2048),
        # the backward pass of the same kind of batch, with the weights' gradients
        _norm("norm backward 4096x1024", "backward", 4096, 1024),
        # rows of an odd length, as no vector load likes them
        _norm("norm backward 5003x1537", "backward", 5003, 1537),
        # the end of a sublayer in training: dropout and the residual sum
        _drop("dropout+residual 4096x1024", "forward", 4096 * 1024, 0.1, 0),
        # its backward pass over a large array of odd length, late in a run (the offset has passed 32 bits)
        _drop("dropout backward odd", "backward", 4093 * 4099, 0.5, 5 << 32),
        # one token being generated: the weights have to be read
        _gated("gated 1 token", "serve", 1, 1024, 4096, "silu"),
        # a few sequences decoded together, no round extent
        _gated("gated 24 tokens ragged", "serve", 24, 1000, 2731, "gelu"),
        # a training batch, forward and backward
        _gated("gated 4096x1024x4096", "train", 4096, 1024, 4096, "silu"),
        _gated("gated backward 4096x1024", "backward", 4096, 1024, 4096, "silu"),
        # a small ragged batch, backward
        _gated("gated backward ragged", "backward", 777, 1000, 1537, "gelu"),
        # the three together with the down projection: forward and backward of a sublayer, all gradients
        _sublayer("sublayer 2048x512x2048", 2048, 512, 2048, 0.1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges: rows from one token to a large batch, widths of any length."""
    kind = rng.choice(["norm", "norm", "drop", "gated", "gated", "gated", "sublayer"])
    if kind == "norm":
        cols = _log_int(rng, 16, 16384)
        case = _norm("", rng.choice(["forward", "backward"]), _log_int(rng, 1, min(65536, (1 << 24) // cols)), cols)
    elif kind == "drop":
        case = _drop("", rng.choice(["forward", "backward"]), _log_int(rng, 1, 1 << 24),
                     round(rng.uniform(0.0, 0.9), 3), rng.randrange(1 << 40))
    else:
        width, inner = _log_int(rng, 32, 4096), _log_int(rng, 32, 8192)
        most = min(8192, 4096 * 1024 * 4096 // (width * inner))
        if kind == "gated":
            case = _gated("", rng.choice(["serve", "train", "backward"]), _log_int(rng, 1, most), width, inner,
                          rng.choice(["silu", "gelu", "relu", "sigmoid"]))
        else:
            case = _sublayer("", _log_int(rng, 1, max(1, most // 2)), width, inner, rng.choice([0.0, 0.1, 0.2]))
    del case["name"]
    return case


# ------------------------------------------------------------------------------- preparing

SEED = 0x1234567890ABCDEF   # of the dropout masks; a program draws one at its start


def _inputs(case, seed):
    """What the path meets: hidden states whose features differ in scale and mean, weights of variance 1 / fan-in,
    gradients that differ from token to token."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def hidden(rows, cols):
        return normal(rows, cols) * torch.exp(0.5 * normal(cols)) + 0.3 * normal(cols)

    def gradient(rows, cols):
        return normal(rows, cols) * torch.exp(normal(rows, 1)) * 1e-3

    def weight(rows, cols):
        return normal(rows, cols) / math.sqrt(rows)

    kind = case["kind"]
    if kind == "norm":
        t = {"x": hidden(case["rows"], case["cols"]), "gamma": 1 + 0.2 * normal(case["cols"]),
             "beta": 0.1 * normal(case["cols"])}
        if case["direction"] == "backward":
            t["dy"] = gradient(case["rows"], case["cols"])
    elif kind == "drop":
        t = {"x": normal(case["count"])}
        if case["direction"] == "forward":
            t["residual"] = normal(case["count"])
    else:
        m, k, f = case["rows"], case["width"], case["inner"]
        t = {"x": normal(m, k) if kind == "gated" else hidden(m, k), "gate": weight(k, f), "up": weight(k, f)}
        if kind == "sublayer":
            t.update(gamma=1 + 0.2 * normal(k), beta=0.1 * normal(k), down=weight(f, k), dy=gradient(m, k))
        elif case["direction"] == "backward":
            # the projections that the forward pass left
            t["pre"] = torch.stack([t["x"] @ t["gate"], t["x"] @ t["up"]])
            t["dh"] = gradient(m, f)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    if own:
        return _own_state(case, t)
    return {"case": case, "t": t}


# ------------------------------------------------------------------- the package's operators

_library = None


def _own_library():
    """The package, and the one stream and handle of a program that calls operators itself."""
    global _library
    if _library is None:
        from tinyflow_amd import gpu_op, ndarray
        stream = gpu_op.create_cudaStream()
        _library = gpu_op, ndarray, stream, gpu_op.create_cublasHandle(stream)
    return _library


class _DeviceView(object):
    """A device array of the library as torch sees foreign device memory."""

    def __init__(self, arr):
        self.__cuda_array_interface__ = {"shape": arr.shape, "typestr": "<f4", "version": 2,
                                         "data": (arr.handle.contents.data, False)}


def _own_state(case, t):
    """The same inputs in the package's arrays, and the arrays that the results go to."""
    _, ndarray, _, _ = _own_library()
    views = {}

    def empty(name, *shape):
        arr = ndarray.empty(shape, ctx=ndarray.gpu(0))
        views[name] = torch.as_tensor(_DeviceView(arr), device="cuda")
        return arr

    a = {}
    for name, value in t.items():
        a[name] = empty(name, *value.shape)
        views[name].copy_(value)
    kind = case["kind"]
    if kind == "norm":
        if case["direction"] == "forward":
            results = {"y": t["x"].shape}
        else:
            results = {"dx": t["x"].shape, "dgamma": t["gamma"].shape, "dbeta": t["beta"].shape}
    elif kind == "drop":
        results = {"y": t["x"].shape}
    else:
        m, k, f = case["rows"], case["width"], case["inner"]
        if kind == "sublayer":
            results = {"y": (m, k), "dx": (m, k), "dgamma": (k,), "dbeta": (k,), "dgate": (k, f), "dup": (k, f),
                       "ddown": (f, k)}
            for name, shape in (("n", (m, k)), ("pre", (2, m, f)), ("h", (m, f)), ("o", (m, k)), ("do", (m, k)),
                                ("dh", (m, f)), ("dn", (m, k)), ("dnorm", (m, k))):
                a[name] = empty(name, *shape)
        elif case["direction"] == "backward":
            results = {"dx": (m, k), "dgate": (k, f), "dup": (k, f)}
        else:
            results = {"h": (m, f)}
            if case["direction"] == "train":
                results["pre"] = (2, m, f)
    for name, shape in results.items():
        a[name] = empty(name, *shape)
    torch.cuda.synchronize()
    return {"case": case, "a": a, "out": {name: views[name] for name in results}}


def _room(wanted):
    if wanted:
        raise MemoryError("%d bytes of device scratch could not be had" % wanted)


def _run_own(state):
    op, _, stream, blas = _own_library()
    case, a = state["case"], state["a"]
    kind = case["kind"]
    if kind == "norm":
        if case["direction"] == "forward":
            op.layer_norm_forward(a["x"], a["gamma"], a["beta"], a["y"], EPS, stream)
        else:
            _room(op.layer_norm_backward(a["x"], a["gamma"], a["dy"], a["dx"], a["dgamma"], a["dbeta"], EPS, stream))
    elif kind == "drop":
        op.counter_dropout(a["x"], a.get("residual"), a["y"], case["dropout"], SEED, case["offset"], stream)
    elif kind == "gated":
        if case["direction"] == "backward":
            _room(op.gated_feed_forward_backward(a["x"], a["gate"], a["up"], a["pre"], a["dh"], a["dx"], a["dgate"],
                                                 a["dup"], case["activation"], stream))
        else:
            _room(op.gated_feed_forward(a["x"], a["gate"], a["up"], a.get("pre"), a["h"], case["activation"], stream))
    else:
        p = case["dropout"]
        op.layer_norm_forward(a["x"], a["gamma"], a["beta"], a["n"], EPS, stream)
        _room(op.gated_feed_forward(a["n"], a["gate"], a["up"], a["pre"], a["h"], "silu", stream))
        op.matrix_multiply(a["h"], False, a["down"], False, a["o"], blas, stream)
        op.counter_dropout(a["o"], a["x"], a["y"], p, SEED, 0, stream)
        op.counter_dropout(a["dy"], None, a["do"], p, SEED, 0, stream)
        op.matrix_multiply(a["h"], True, a["do"], False, a["ddown"], blas, stream)
        op.matrix_multiply(a["do"], False, a["down"], True, a["dh"], blas, stream)
        _room(op.gated_feed_forward_backward(a["n"], a["gate"], a["up"], a["pre"], a["dh"], a["dn"], a["dgate"],
                                             a["dup"], "silu", stream))
        _room(op.layer_norm_backward(a["x"], a["gamma"], a["dn"], a["dnorm"], a["dgamma"], a["dbeta"], EPS, stream))
        op.matrix_elementwise_add(a["dnorm"], a["dy"], a["dx"], stream)
    return state["out"]


# ---------------------------------------------------------------------------- the plain form

def _statistics(x):
    centred = x - x.mean(1, keepdim=True)
    return centred, torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPS)


def _plain_norm(x, gamma, beta):
    centred, inverse = _statistics(x)
    return centred * inverse * gamma + beta


def _plain_norm_backward(x, gamma, dy):
    centred, inverse = _statistics(x)
    normed, scaled = centred * inverse, dy * gamma
    dx = inverse * (scaled - scaled.mean(1, keepdim=True) - normed * (scaled * normed).mean(1, keepdim=True))
    return dx, (dy * normed).sum(0), dy.sum(0)


def _plain_activation(g, activation):
    """(act(g), act'(g))"""
    if activation == "relu":
        return torch.clamp(g, min=0), (g > 0).float()
    if activation == "gelu":
        phi = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-g))
    if activation == "sigmoid":
        return s, s * (1 - s)
    return g * s, s * (1 + g * (1 - s))


def _plain_gated(x, gate, up, activation):
    g, u = x @ gate, x @ up
    return g, u, _plain_activation(g, activation)[0] * u


def _plain_gated_backward(x, gate, up, g, u, dh, activation):
    act, slope = _plain_activation(g, activation)
    dg, du = dh * u * slope, dh * act
    return dg @ gate.t() + du @ up.t(), x.t() @ dg, x.t() @ du


def _high_low(factor, c):
    """The high and the low 32 bits of factor * c for words held in 64-bit integers."""
    high, low = factor * (c >> 16), factor * (c & 0xFFFF)
    return (high + (low >> 16)) >> 16, ((high << 16) + low) & 0xFFFFFFFF


def _plain_words(count, seed, offset):
    block = torch.arange((count + 3) // 4, device="cuda")
    c0, c1 = block & 0xFFFFFFFF, block >> 32
    c2, c3 = torch.full_like(block, offset & 0xFFFFFFFF), torch.full_like(block, offset >> 32)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        h0, l0 = _high_low(0xD2511F53, c0)
        h1, l1 = _high_low(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack([c0, c1, c2, c3], 1).reshape(-1)[:count]


def _threshold_scale(dropout):
    p = np.float32(dropout)
    return int(float(p) * 2.0 ** 32), float(np.float32(1) / (np.float32(1) - p))


def _plain_dropout(x, dropout, offset):
    threshold, scale = _threshold_scale(dropout)
    keep = (_plain_words(x.numel(), SEED, offset) >= threshold).reshape(x.shape)
    return torch.where(keep, x * scale, torch.zeros_like(x))


def _run_plain(state):
    case, t = state["case"], state["t"]
    kind = case["kind"]
    if kind == "norm":
        if case["direction"] == "forward":
            return {"y": _plain_norm(t["x"], t["gamma"], t["beta"])}
        return dict(zip(("dx", "dgamma", "dbeta"), _plain_norm_backward(t["x"], t["gamma"], t["dy"])))
    if kind == "drop":
        y = _plain_dropout(t["x"], case["dropout"], case["offset"])
        return {"y": y + t["residual"] if "residual" in t else y}
    if kind == "gated":
        if case["direction"] == "backward":
            return dict(zip(("dx", "dgate", "dup"),
                            _plain_gated_backward(t["x"], t["gate"], t["up"], t["pre"][0], t["pre"][1], t["dh"],
                                                  case["activation"])))
        g, u, h = _plain_gated(t["x"], t["gate"], t["up"], case["activation"])
        return {"h": h, "pre": torch.stack([g, u])} if case["direction"] == "train" else {"h": h}
    n = _plain_norm(t["x"], t["gamma"], t["beta"])
    g, u, h = _plain_gated(n, t["gate"], t["up"], "silu")
    y = t["x"] + _plain_dropout(h @ t["down"], case["dropout"], 0)
    do = _plain_dropout(t["dy"], case["dropout"], 0)
    dn, dgate, dup = _plain_gated_backward(n, t["gate"], t["up"], g, u, do @ t["down"].t(), "silu")
    dx, dgamma, dbeta = _plain_norm_backward(t["x"], t["gamma"], dn)
    return {"y": y, "dx": dx + t["dy"], "dgamma": dgamma, "dbeta": dbeta, "dgate": dgate, "dup": dup,
            "ddown": h.t() @ do}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------- in 64 bits

def _exact_mask(count, seed, offset, dropout):
    """The kept elements' factor, by numpy on unsigned words."""
    low = np.uint64(0xFFFFFFFF)
    block = np.arange((count + 3) // 4, dtype=np.uint64)
    c = [block & low, block >> np.uint64(32), np.full_like(block, offset & 0xFFFFFFFF), np.full_like(block, offset >> 32)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p, q = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(q >> np.uint64(32)) ^ c[1] ^ np.uint64(key[0]), q & low,
             (p >> np.uint64(32)) ^ c[3] ^ np.uint64(key[1]), p & low]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    words = np.stack(c, axis=1).ravel()[:count]
    kept = words >= np.uint64(math.floor(float(np.float32(dropout)) * 2 ** 32))
    return torch.from_numpy(kept).cuda().double() / (1.0 - float(np.float32(dropout)))


def _exact_norm(x, gamma, beta):
    mean = x.sum(1, keepdim=True) / x.shape[1]
    variance = ((x - mean) ** 2).sum(1, keepdim=True) / x.shape[1]
    return gamma * ((x - mean) / (variance + EPS) ** 0.5) + beta


def _exact_act(g, activation):
    if activation == "relu":
        return g * (g > 0)
    if activation == "gelu":
        return g * torch.special.ndtr(g)
    return torch.sigmoid(g) * (g if activation == "silu" else 1)


def exact(case, seed):
    """The definitions in 64 bits; gradients by differentiating them."""
    t = {name: v.double() for name, v in _inputs(case, seed).items()}
    kind = case["kind"]
    if kind == "drop":
        y = t["x"] * _exact_mask(case["count"], SEED, case["offset"], case["dropout"])
        return {"y": y + t["residual"] if "residual" in t else y}
    if kind == "norm":
        if case["direction"] == "forward":
            return {"y": _exact_norm(t["x"], t["gamma"], t["beta"])}
        wrt = [t[n].requires_grad_() for n in ("x", "gamma", "beta")]
        found = torch.autograd.grad(_exact_norm(*wrt), wrt, t["dy"])
        return dict(zip(("dx", "dgamma", "dbeta"), found))
    if kind == "gated":
        if case["direction"] != "backward":
            g, u = t["x"] @ t["gate"], t["x"] @ t["up"]
            h = _exact_act(g, case["activation"]) * u
            return {"h": h, "pre": torch.stack([g, u])} if case["direction"] == "train" else {"h": h}
        # the projections are inputs here, as the forward pass rounded them
        pre = t["pre"].requires_grad_()
        dg, du = torch.autograd.grad(_exact_act(pre[0], case["activation"]) * pre[1], pre, t["dh"])[0]
        return {"dx": dg @ t["gate"].t() + du @ t["up"].t(), "dgate": t["x"].t() @ dg, "dup": t["x"].t() @ du}
    names = ("x", "gamma", "beta", "gate", "up", "down")
    for name in names:
        t[name].requires_grad_()
    n = _exact_norm(t["x"], t["gamma"], t["beta"])
    h = _exact_act(n @ t["gate"], "silu") * (n @ t["up"])
    mask = _exact_mask(t["x"].numel(), SEED, 0, case["dropout"]).reshape(t["x"].shape)
    y = t["x"] + h @ t["down"] * mask
    found = torch.autograd.grad(y, [t[name] for name in names], t["dy"])
    return dict({"d" + name: v for name, v in zip(names, found)}, y=y.detach())


# ---------------------------------------------------------------------- what it has to cost

def work(case):
    """Each input read once and each output written once; the products' multiply-adds, and a handful of operations an
    element elsewhere."""
    kind = case["kind"]
    if kind == "norm":
        n, c = case["rows"] * case["cols"], case["cols"]
        if case["direction"] == "forward":
            return {"bytes": 4 * (2 * n + 2 * c), "flops": 8 * n}
        return {"bytes": 4 * (3 * n + 3 * c), "flops": 18 * n}
    if kind == "drop":
        return {"bytes": 4 * case["count"] * (3 if case["direction"] == "forward" else 2), "flops": 2 * case["count"]}
    m, k, f = case["rows"], case["width"], case["inner"]
    if kind == "gated":
        if case["direction"] == "backward":
            return {"bytes": 4 * (2 * m * k + 4 * k * f + 3 * m * f), "flops": 12 * m * k * f}
        return {"bytes": 4 * (m * k + 2 * k * f + m * f * (3 if case["direction"] == "train" else 1)),
                "flops": 4 * m * k * f}
    # between the two passes the projections and their product (3 m f) are written and read
    return {"bytes": 4 * (4 * m * k + 6 * k * f + 6 * m * f + 4 * k), "flops": 18 * m * k * f}
