"""The operators of an attention sublayer, y = x + attention(rotated(q), rotated(k), v) W, as cases that can be timed: the
norm, rotation and placement of heads, attention of few queries over a long cache, attention of whole sequences, each of the
last forward and backward, and a run of them together.

``own`` false: the operators in plain torch, fp32 (angles in 64 bits). ``own`` true: the calls that a user makes of
``tinyflow_amd.gpu_op``. Everything is fp32, the one type of the package's arrays.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
NORM_EPS = 1e-5   # of the layer norm in front of the sublayer


# ------------------------------------------------------------------------------ the cases

def _heads(name, direction, rows, heads, key_heads, dim, rotary, interleaved, first, capacity=0):
    """``serve`` places keys and values in a cache of ``capacity`` rows; ``forward`` and ``backward`` norm and rotate queries
    and keys in place of their rows. Positions count from ``first``."""
    return {"name": name, "kind": "heads", "direction": direction, "rows": rows, "heads": heads, "key_heads": key_heads,
            "dim": dim, "rotary": rotary, "interleaved": interleaved, "first": first, "capacity": capacity}


def _cache(name, batch, queries, keys, longest, heads, key_heads, dim, cap, distance):
    """``queries`` new tokens of each sequence against a cache of ``keys`` rows, of which the longest sequence has used ``longest``."""
    return {"name": name, "kind": "cache", "batch": batch, "queries": queries, "keys": keys, "longest": longest,
            "heads": heads, "key_heads": key_heads, "dim": dim, "cap": cap, "distance": distance}


def _attention(name, direction, mask, batch, tokens, heads, key_heads, dim, cap, distance):
    """``serve``: the output alone; ``train``: with the statistics that the backward pass reads; ``backward``."""
    return {"name": name, "kind": "attention", "direction": direction, "mask": mask, "batch": batch, "tokens": tokens,
            "heads": heads, "key_heads": key_heads, "dim": dim, "cap": cap, "distance": distance}


def _sublayer(name, mask, batch, tokens, width, heads, key_heads, dim):
    return {"name": name, "kind": "sublayer", "mask": mask, "batch": batch, "tokens": tokens, "width": width, "heads": heads,
            "key_heads": key_heads, "dim": dim, "cap": 0.0, "distance": False}


def listed():
    return [
        # one token being generated: its queries, keys and values, the latter two to the cache
        _heads("heads 1 token", "serve", 1, 16, 4, 128, 128, False, 2047, 4096),
        # the tokens of a training batch
        _heads("heads 4096x16+4x128", "forward", 4096, 16, 4, 128, 128, False, 0),
        _heads("heads backward 4096x16+4x128", "backward", 4096, 16, 4, 128, 128, False, 0),
        # the end of a very long context: half of a head is rotated, in pairs of neighbours, at positions past a million
        _heads("heads backward ragged far", "backward", 1531, 6, 3, 80, 40, True, 1 << 20),
        # eight sequences decoded together, of unlike lengths
        _cache("cache 8 sequences", 8, 1, 8192, 8192, 16, 4, 128, 0.0, False),
        # one long sequence
        _cache("cache 100003", 1, 1, 131072, 100003, 16, 2, 128, 0.0, False),
        # a few tokens checked at once against a short cache, scores capped, biased by distance: latency
        _cache("cache 5 tokens ragged", 2, 5, 1500, 1237, 8, 8, 64, 30.0, True),
        # prompts read in, no gradient
        _attention("prompt 2x2048", "serve", "causal", 2, 2048, 16, 4, 64, 0.0, False),
        # a training sequence, forward and backward
        _attention("attention 4096x16x128", "train", "causal", 1, 4096, 16, 4, 128, 0.0, False),
        _attention("attention backward 4096x16x128", "backward", "causal", 1, 4096, 16, 4, 128, 0.0, False),
        # packed documents of unlike lengths, no round extent, capped scores with a bias by distance
        _attention("attention backward ragged", "backward", "documents", 2, 1777, 6, 3, 72, 20.0, True),
        # all of it: forward and backward of a sublayer whose sequences see a prefix in both directions, all gradients
        _sublayer("sublayer 4x1024x1024", "prefix", 4, 1024, 1024, 16, 4, 64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges: one token to long sequences, heads of any length, alone and shared."""
    kind = rng.choice(["heads", "heads", "cache", "cache", "attention", "attention", "attention", "sublayer"])
    key_heads = rng.choice([1, 2, 3, 4, 8])
    heads = key_heads * rng.choice([1, 1, 2, 4, 7])
    dim = rng.choice([64, 128, _log_int(rng, 16, 256)])
    cap, distance = rng.choice([0.0, 0.0, 30.0]), rng.random() < 0.25
    if kind == "heads":
        dim += dim % 2
        rotary = rng.choice([dim, 2 * rng.randint(1, dim // 2)])
        direction = rng.choice(["serve", "forward", "backward"])
        rows = _log_int(rng, 1, min(16384, (1 << 23) // (heads * dim)))
        if direction == "serve":
            rows = min(rows, 64)
        case = _heads("", direction, rows, heads, key_heads, dim, rotary, rng.random() < 0.5, rng.choice([0, _log_int(rng, 1, 1 << 22)]),
                      rows + _log_int(rng, 1, 4096) if direction == "serve" else 0)
    elif kind == "cache":
        batch = _log_int(rng, 1, 32)
        queries = rng.choice([1, 1, 1, rng.randint(2, 8)])
        keys = queries + _log_int(rng, 1, min(131072, (3 << 23) // (batch * key_heads * dim)))
        case = _cache("", batch, queries, keys, rng.randint(max(queries, keys // 2), keys), heads, key_heads, dim, cap, distance)
    else:
        mask = rng.choice(["causal", "documents", "prefix", "full"])
        batch = _log_int(rng, 1, 4)
        # the causal 4096 tokens of 16 heads of 128 columns, and no more
        most = math.sqrt(4096 * 4096 * 16 * 128 / (2 * batch * heads * dim))
        if kind == "attention":
            direction = rng.choice(["serve", "train", "backward"])
            # (the gradients of a few tokens' scores are nothing but rounding)
            tokens = _log_int(rng, 32 if direction == "backward" else 1, min(8192, int(most)))
            case = _attention("", direction, mask, batch, tokens, heads, key_heads, dim, cap, distance)
        else:
            dim += dim % 2
            width = _log_int(rng, 32, 1024)
            most = min(1024, most / 2, 8192 * 1024 * 1024 / (batch * width * (heads + key_heads) * dim))
            case = _sublayer("", mask, batch, _log_int(rng, 32, int(most)), width, heads, key_heads, dim)
    del case["name"]
    return case


# ------------------------------------------------------------------------------- preparing

def _shares(total, parts):
    """``total`` in ``parts`` unlike parts, the last ones several times the first."""
    parts = max(1, min(parts, total))
    ends = [total * i * (i + 1) // (parts * (parts + 1)) for i in range(parts + 1)]
    sizes = [b - a for a, b in zip(ends, ends[1:])]
    return [s for s in sizes if s] or [total]


def _lengths(case):
    """How much of the cache each sequence has used, its new tokens among it."""
    b, q = case["batch"], case["queries"]
    return [q + (case["longest"] - q) * (i + 1) // b for i in range(b)]


def _prefixes(case):
    b = case["batch"]
    return [case["tokens"] * (i + 1) // (2 * b) for i in range(b)]


def _spans(case, rng):
    """[batch, queries, 2]: the first key that a query sees and the one behind the last; None where ``causal`` says it all."""
    if case["kind"] == "cache":
        q = case["queries"]
        lengths = np.array(_lengths(case))[rng.permutation(case["batch"])]
        last = lengths[:, None] - q + 1 + np.arange(q)
        return np.stack([np.zeros_like(last), last], 2)
    b, t = case["batch"], case["tokens"]
    at = np.arange(t)
    if case["mask"] == "documents":
        spans = []
        for _ in range(b):
            sizes = np.array(_shares(t, 4))
            sizes = sizes[rng.permutation(len(sizes))]
            starts = np.repeat(np.cumsum(sizes) - sizes, sizes)
            spans.append(np.stack([starts, at + 1], 1))
        return np.stack(spans)
    if case["mask"] == "prefix":
        prefixes = np.array(_prefixes(case))[rng.permutation(b)]
        return np.stack([np.zeros((b, t), int), np.maximum(prefixes[:, None], at + 1)], 2)
    return None


def _pairs(case):
    """Pairs of a query and a key that it sees, of one head."""
    if case["kind"] == "cache":
        q = case["queries"]
        return sum(n * q - q * (q - 1) // 2 for n in _lengths(case))
    b, t = case["batch"], case["tokens"]
    if case["mask"] == "documents":
        return b * sum(n * (n + 1) // 2 for n in _shares(t, 4))
    if case["mask"] == "prefix":
        return sum(t * (t + 1) // 2 + p * (p - 1) // 2 for p in _prefixes(case))
    return b * (t * (t + 1) // 2 if case["mask"] == "causal" else t * t)


def _frequencies(rotary):
    """Slow ones four times slower for a longer context, fast ones as they were, those between by parts."""
    i = np.arange(rotary // 2)
    f = 10000.0 ** (-2.0 * i / rotary)
    turns = 2048 * f / (2 * math.pi)   # over the shorter context
    kept = np.clip((turns - 1) / (32 - 1), 0, 1)
    return (f * (kept + (1 - kept) / 4)).astype(np.float32)


AMPLITUDE = 1 + 0.1 * math.log(4)   # of rotated columns, for the same context


def _slopes(heads):
    return (2.0 ** (-8.0 * (np.arange(heads) + 1) / heads)).astype(np.float32)


def _inputs(case, seed):
    """What the path meets: projections whose columns differ in scale, weights of variance 1 / fan-in, gradients that differ
    from token to token."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 32))

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def device(values):
        return torch.as_tensor(np.ascontiguousarray(values, np.float32)).cuda()

    def gradient(rows, cols):
        return normal(rows, cols) * torch.exp(normal(rows, 1)) * 1e-3

    kind, h, hk, d = case["kind"], case["heads"], case["key_heads"], case["dim"]
    if kind == "heads":
        n = case["rows"]
        t = {"q": normal(n, h * d) * torch.exp(0.5 * normal(h * d)), "k": normal(n, hk * d) * torch.exp(0.5 * normal(hk * d)),
             "gq": 1 + 0.2 * normal(d), "gk": 1 + 0.2 * normal(d), "frequencies": device(_frequencies(case["rotary"])),
             "positions": device(case["first"] + np.arange(n))}
        if case["direction"] == "serve":
            # the rows behind what the sequence has used
            used = case["capacity"] - n
            t.update(v=normal(n, hk * d), slots=device((used + np.arange(n))[None, :]),
                     k_cache=normal(1, case["capacity"], hk * d), v_cache=normal(1, case["capacity"], hk * d))
        elif case["direction"] == "backward":
            t.update(dq=gradient(n, h * d), dk=gradient(n, hk * d))
        return t
    if kind == "sublayer":
        b, n, w = case["batch"], case["tokens"], case["width"]
        t = {"x": normal(b * n, w) * torch.exp(0.5 * normal(w)) + 0.3 * normal(w), "gamma": 1 + 0.2 * normal(w),
             "beta": 0.1 * normal(w), "wq": normal(w, h * d) / math.sqrt(w), "wk": normal(w, hk * d) / math.sqrt(w),
             "wv": normal(w, hk * d) / math.sqrt(w), "wo": normal(h * d, w) / math.sqrt(h * d), "gq": 1 + 0.2 * normal(d),
             "gk": 1 + 0.2 * normal(d), "frequencies": device(_frequencies(d)), "positions": device(np.arange(n)),
             "dy": gradient(b * n, w)}
    else:
        b = case["batch"]
        tq, tk = (case["queries"], case["keys"]) if kind == "cache" else (case["tokens"], case["tokens"])
        # queries and keys as their norms leave them
        t = {"q": 1.5 * normal(b, tq, h, d), "k": normal(b, tk, hk, d), "v": normal(b, tk, hk, d) * torch.exp(0.5 * normal(hk, d))}
        if case["distance"]:
            t["slopes"] = device(_slopes(h))
    spans = _spans(case, rng)
    if spans is not None:
        t["spans"] = device(spans)
    if kind == "attention" and case["direction"] == "backward":
        t["out"], t["stat"] = _plain_attention(t["q"], t["k"], t["v"], t.get("spans"), t.get("slopes"), _scale(case), case["cap"],
                                               case["mask"] == "causal")
        t["do"] = normal(b, tq, h, d) * torch.exp(normal(b, tq, 1, 1)) * 1e-3
    return t


def _scale(case):
    return 1 / math.sqrt(case["dim"])


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
    kind, h, hk, d = case["kind"], case["heads"], case["key_heads"], case["dim"]
    results, kept = {}, []
    if kind == "heads":
        if case["direction"] == "backward":
            results = {"dq_in": t["q"].shape, "dk_in": t["k"].shape, "dgq": (d,), "dgk": (d,)}
        else:
            results = {"q_out": t["q"].shape}
            if case["direction"] == "forward":
                results["k_out"] = t["k"].shape
            else:
                kept = ["k_cache", "v_cache"]
    elif kind == "sublayer":
        rows, w = t["x"].shape[0], case["width"]
        results = {"y": (rows, w), "dx": (rows, w), "dgamma": (w,), "dbeta": (w,), "dwq": (w, h * d), "dwk": (w, hk * d),
                   "dwv": (w, hk * d), "dwo": (h * d, w), "dgq": (d,), "dgk": (d,)}
        for name in ("n", "p", "dn", "dn_k", "dn_v"):
            a[name] = empty(name, rows, w)
        for name in ("q", "q_rot", "att", "dq", "datt", "dq_rot"):
            a[name] = empty(name, rows, h * d)
        for name in ("k", "k_rot", "v", "dk", "dv", "dk_rot"):
            a[name] = empty(name, rows, hk * d)
        a["stat"] = empty("stat", case["batch"], h, case["tokens"])
    elif kind == "attention" and case["direction"] == "backward":
        results = {"dq": t["q"].shape, "dk": t["k"].shape, "dv": t["v"].shape}
    else:
        results = {"out": t["q"].shape}
        if kind == "attention" and case["direction"] == "train":
            results["stat"] = (case["batch"], h, case["tokens"])
    for name, shape in results.items():
        a[name] = empty(name, *shape)
    torch.cuda.synchronize()
    return {"case": case, "a": a, "out": {name: views[name] for name in list(results) + kept}, "views": views}


def _room(wanted):
    if wanted:
        raise MemoryError("%d bytes of device scratch could not be had" % wanted)


def _run_own(state):
    op, _, stream, blas = _own_library()
    case, a = state["case"], state["a"]
    kind, h, hk = case["kind"], case["heads"], case["key_heads"]
    if kind == "heads":
        turn = a["positions"], a["frequencies"], AMPLITUDE, case["interleaved"]
        if case["direction"] == "backward":
            _room(op.head_rotary_backward([op.head_gradient_part(a["q"], a["gq"], a["dq"], a["dq_in"], a["dgq"], h),
                                           op.head_gradient_part(a["k"], a["gk"], a["dk"], a["dk_in"], a["dgk"], hk)],
                                          *turn, EPS, stream))
        elif case["direction"] == "forward":
            op.head_rotary([op.head_part(a["q"], a["gq"], a["q_out"], h), op.head_part(a["k"], a["gk"], a["k_out"], hk)],
                           *turn, EPS, None, stream)
        else:
            op.head_rotary([op.head_part(a["q"], a["gq"], a["q_out"], h),
                            op.head_part(a["k"], a["gk"], a["k_cache"], hk, place=True),
                            op.head_part(a["v"], None, a["v_cache"], hk, rotate=False, place=True)],
                           *turn, EPS, a["slots"], stream)
    elif kind == "sublayer":
        _sublayer_own(op, stream, blas, case, a)
    else:
        shared = case["batch"], h, hk, _scale(case), case["cap"], kind == "attention" and case["mask"] == "causal"
        inputs = a["q"], a["k"], a["v"], a.get("spans"), a.get("slopes")
        if kind == "attention" and case["direction"] == "backward":
            _room(op.attention_backward(*inputs, a["out"], a["stat"], a["do"], a["dq"], a["dk"], a["dv"], *shared, stream))
        else:
            _room(op.attention_forward(*inputs, a["out"], a.get("stat"), *shared, stream))
    return state["out"]


def _sublayer_own(op, stream, blas, case, a):
    h, hk = case["heads"], case["key_heads"]
    turn = a["positions"], a["frequencies"], 1.0, False
    shared = case["batch"], h, hk, _scale(case), 0.0, case["mask"] == "causal"

    def multiply(x, tx, y, ty, out):
        op.matrix_multiply(x, tx, y, ty, out, blas, stream)
    op.layer_norm_forward(a["x"], a["gamma"], a["beta"], a["n"], NORM_EPS, stream)
    for w, out in (("wq", "q"), ("wk", "k"), ("wv", "v")):
        multiply(a["n"], False, a[w], False, a[out])
    op.head_rotary([op.head_part(a["q"], a["gq"], a["q_rot"], h), op.head_part(a["k"], a["gk"], a["k_rot"], hk)],
                   *turn, EPS, None, stream)
    inputs = a["q_rot"], a["k_rot"], a["v"], a.get("spans"), None
    _room(op.attention_forward(*inputs, a["att"], a["stat"], *shared, stream))
    multiply(a["att"], False, a["wo"], False, a["p"])
    op.matrix_elementwise_add(a["p"], a["x"], a["y"], stream)
    multiply(a["att"], True, a["dy"], False, a["dwo"])
    multiply(a["dy"], False, a["wo"], True, a["datt"])
    _room(op.attention_backward(*inputs, a["att"], a["stat"], a["datt"], a["dq_rot"], a["dk_rot"], a["dv"], *shared, stream))
    _room(op.head_rotary_backward([op.head_gradient_part(a["q"], a["gq"], a["dq_rot"], a["dq"], a["dgq"], h),
                                   op.head_gradient_part(a["k"], a["gk"], a["dk_rot"], a["dk"], a["dgk"], hk)],
                                  *turn, EPS, stream))
    for w, d, dn in (("wq", "dq", "dn"), ("wk", "dk", "dn_k"), ("wv", "dv", "dn_v")):
        multiply(a["n"], True, a[d], False, a["d" + w])
        multiply(a[d], False, a[w], True, a[dn])
    op.matrix_elementwise_add(a["dn"], a["dn_k"], a["dn"], stream)
    op.matrix_elementwise_add(a["dn"], a["dn_v"], a["dn"], stream)
    _room(op.layer_norm_backward(a["x"], a["gamma"], a["dn"], a["p"], a["dgamma"], a["dbeta"], NORM_EPS, stream))
    op.matrix_elementwise_add(a["p"], a["dy"], a["dx"], stream)


# ---------------------------------------------------------------------------- the plain form

def _plain_turn(positions, frequencies, rows):
    """Cosines and sines [rows, 1, rotary / 2], from angles in 64 bits."""
    angles = positions.double().reshape(-1)[:, None] * frequencies.double()
    angles = angles.repeat(rows // angles.shape[0], 1)[:, None, :]
    return torch.cos(angles).float(), torch.sin(angles).float()


def _plain_rotate(x, cos, sin, interleaved, amplitude):
    """x [rows, heads, dim]"""
    r = 2 * cos.shape[2]
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
    u, w = (a * cos - b * sin) * amplitude, (a * sin + b * cos) * amplitude
    turned = torch.stack([u, w], 3).flatten(2) if interleaved else torch.cat([u, w], 2)
    return torch.cat([turned, x[..., r:]], 2)


def _plain_heads(x, gamma, heads, cos, sin, interleaved, amplitude):
    rows = x.shape[0]
    y = x.reshape(rows, heads, -1)
    y = y * torch.rsqrt((y * y).mean(2, keepdim=True) + EPS) * gamma
    return _plain_rotate(y, cos, sin, interleaved, amplitude).reshape(rows, -1)


def _plain_heads_backward(x, gamma, dy, heads, cos, sin, interleaved, amplitude):
    rows = x.shape[0]
    x, dy = x.reshape(rows, heads, -1), dy.reshape(rows, heads, -1)
    da = _plain_rotate(dy, cos, -sin, interleaved, amplitude)
    inverse = torch.rsqrt((x * x).mean(2, keepdim=True) + EPS)
    normed, scaled = x * inverse, da * gamma
    dx = inverse * (scaled - normed * (scaled * normed).mean(2, keepdim=True))
    return dx.reshape(rows, -1), (da * normed).sum((0, 1))


def _plain_seen(tq, tk, spans, causal):
    """[batch or 1, 1, queries, keys]"""
    at = torch.arange(tk, device="cuda", dtype=torch.float32)
    seen = torch.ones(1, 1, tq, tk, device="cuda", dtype=torch.bool)
    if spans is not None:
        seen = ((at >= spans[:, :, :1]) & (at < spans[:, :, 1:]))[:, None]
    if causal:
        seen = seen & (at <= torch.arange(tk - tq, tk, device="cuda", dtype=torch.float32)[:, None])
    return seen


def _plain_scores(q, k, spans, slopes, scale, cap, causal):
    """Scores [batch, heads, queries, keys], -inf where a query does not see a key, and the slope of the cap."""
    b, tq, h, d = q.shape
    tk, hk = k.shape[1], k.shape[2]
    rows = q.permute(0, 2, 1, 3).reshape(b, hk, h // hk * tq, d)
    s = (rows @ k.permute(0, 2, 3, 1).contiguous()).reshape(b, h, tq, tk) * scale
    slope = None
    if cap:
        s = torch.tanh(s / cap)
        slope = 1 - s * s
        s = s * cap
    if slopes is not None:
        ahead = torch.arange(tk - tq, tk, device="cuda", dtype=torch.float32)[:, None] - torch.arange(tk, device="cuda", dtype=torch.float32)
        s = s - slopes[:, None, None] * ahead.abs()
    return s.masked_fill(~_plain_seen(tq, tk, spans, causal), -math.inf), slope


def _plain_attention(q, k, v, spans, slopes, scale, cap, causal):
    b, tq, h, d = q.shape
    hk = k.shape[2]
    s, _ = _plain_scores(q, k, spans, slopes, scale, cap, causal)
    top = s.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(3, keepdim=True)
    some = total > 0
    out = (p.reshape(b, hk, -1, k.shape[1]) @ v.permute(0, 2, 1, 3).contiguous()).reshape(b, h, tq, d)
    out = out / torch.where(some, total, torch.ones_like(total))
    stat = torch.where(some, top + torch.log(total), torch.full_like(top, -math.inf))
    return out.permute(0, 2, 1, 3).contiguous(), stat[..., 0]


def _plain_attention_backward(q, k, v, out, stat, do, spans, slopes, scale, cap, causal):
    b, tq, h, d = q.shape
    tk, hk = k.shape[1], k.shape[2]

    def by_head(x):
        return x.permute(0, 2, 1, 3).reshape(b, hk, -1, d)

    s, slope = _plain_scores(q, k, spans, slopes, scale, cap, causal)
    p = torch.where(s == -math.inf, torch.zeros_like(s), torch.exp(s - stat[..., None]))
    del s
    delta = (do * out).sum(3).permute(0, 2, 1)[..., None]
    dp = (by_head(do) @ v.permute(0, 2, 3, 1).contiguous()).reshape(b, h, tq, tk)
    ds = p * (dp - delta) * scale
    if cap:
        ds = ds * slope
    del dp
    ds, p = ds.reshape(b, hk, -1, tk), p.reshape(b, hk, -1, tk)
    dq = (ds @ by_head(k)).reshape(b, h, tq, d).permute(0, 2, 1, 3).contiguous()
    dk = (ds.transpose(2, 3) @ by_head(q)).permute(0, 2, 1, 3).contiguous()
    dv = (p.transpose(2, 3) @ by_head(do)).permute(0, 2, 1, 3).contiguous()
    return dq, dk, dv


def _statistics(x):
    centred = x - x.mean(1, keepdim=True)
    return centred, torch.rsqrt((centred * centred).mean(1, keepdim=True) + NORM_EPS)


def _plain_sublayer(case, t):
    b, n, h, hk, d = (case[name] for name in ("batch", "tokens", "heads", "key_heads", "dim"))
    rows, causal = b * n, case["mask"] == "causal"

    def heads_of(x, count):
        return x.reshape(b, n, count, d)
    centred, inverse = _statistics(t["x"])
    normed = centred * inverse
    norm = normed * t["gamma"] + t["beta"]
    q, k, v = norm @ t["wq"], norm @ t["wk"], norm @ t["wv"]
    cos, sin = _plain_turn(t["positions"], t["frequencies"], rows)
    q_rot = heads_of(_plain_heads(q, t["gq"], h, cos, sin, False, 1.0), h)
    k_rot = heads_of(_plain_heads(k, t["gk"], hk, cos, sin, False, 1.0), hk)
    shared = t.get("spans"), None, _scale(case), 0.0, causal
    out, stat = _plain_attention(q_rot, k_rot, heads_of(v, hk), *shared)
    att = out.reshape(rows, -1)
    y = t["x"] + att @ t["wo"]
    dy = t["dy"]
    datt = dy @ t["wo"].t()
    dq, dk, dv = _plain_attention_backward(q_rot, k_rot, heads_of(v, hk), out, stat, heads_of(datt, h), *shared)
    dv = dv.reshape(rows, -1)
    dq, dgq = _plain_heads_backward(q, t["gq"], dq.reshape(rows, -1), h, cos, sin, False, 1.0)
    dk, dgk = _plain_heads_backward(k, t["gk"], dk.reshape(rows, -1), hk, cos, sin, False, 1.0)
    dn = dq @ t["wq"].t() + dk @ t["wk"].t() + dv @ t["wv"].t()
    scaled = dn * t["gamma"]
    dx = inverse * (scaled - scaled.mean(1, keepdim=True) - normed * (scaled * normed).mean(1, keepdim=True))
    return {"y": y, "dx": dx + dy, "dgamma": (dn * normed).sum(0), "dbeta": dn.sum(0), "dwq": norm.t() @ dq,
            "dwk": norm.t() @ dk, "dwv": norm.t() @ dv, "dwo": att.t() @ dy, "dgq": dgq, "dgk": dgk}


def _run_plain(state):
    case, t = state["case"], state["t"]
    kind, h, hk = case["kind"], case["heads"], case["key_heads"]
    if kind == "sublayer":
        return _plain_sublayer(case, t)
    if kind == "heads":
        turn = *_plain_turn(t["positions"], t["frequencies"], case["rows"]), case["interleaved"], AMPLITUDE
        if case["direction"] == "backward":
            dq, dgq = _plain_heads_backward(t["q"], t["gq"], t["dq"], h, *turn)
            dk, dgk = _plain_heads_backward(t["k"], t["gk"], t["dk"], hk, *turn)
            return {"dq_in": dq, "dk_in": dk, "dgq": dgq, "dgk": dgk}
        q = _plain_heads(t["q"], t["gq"], h, *turn)
        k = _plain_heads(t["k"], t["gk"], hk, *turn)
        if case["direction"] == "forward":
            return {"q_out": q, "k_out": k}
        slots = t["slots"][0].long()
        t["k_cache"][0].index_copy_(0, slots, k)
        t["v_cache"][0].index_copy_(0, slots, t["v"])
        return {"q_out": q, "k_cache": t["k_cache"], "v_cache": t["v_cache"]}
    shared = t.get("spans"), t.get("slopes"), _scale(case), case["cap"], kind == "attention" and case["mask"] == "causal"
    if kind == "attention" and case["direction"] == "backward":
        return dict(zip(("dq", "dk", "dv"), _plain_attention_backward(t["q"], t["k"], t["v"], t["out"], t["stat"], t["do"], *shared)))
    out, stat = _plain_attention(t["q"], t["k"], t["v"], *shared)
    return {"out": out, "stat": stat} if kind == "attention" and case["direction"] == "train" else {"out": out}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------- in 64 bits

def _exact_heads(x, gamma, heads, positions, frequencies, interleaved, amplitude):
    """x [rows, heads dim]: the norm, and the rotation as a product of complex numbers."""
    rows, r = x.shape[0], 2 * len(frequencies)
    y = x.reshape(rows, heads, -1)
    if gamma is not None:
        y = y / ((y ** 2).sum(2, keepdim=True) / y.shape[2] + EPS) ** 0.5 * gamma
    angle = torch.outer(positions.reshape(-1).repeat(rows // positions.numel()), frequencies)
    turn = torch.polar(torch.full_like(angle, amplitude), angle)[:, None]
    pairs = y[..., :r].reshape(rows, heads, *((r // 2, 2) if interleaved else (2, r // 2)))
    if not interleaved:
        pairs = pairs.transpose(2, 3)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    turned = (turned if interleaved else turned.transpose(2, 3)).reshape(rows, heads, r)
    return torch.cat([turned, y[..., r:]], 2).reshape(rows, -1)


def _exact_probabilities(q, k, span, slope, scale, cap, causal, stat=None):
    """Of one head: (p, natural logarithm of the sums, derivative of the cap). q [queries, dim], k [keys, dim]"""
    tq, tk = len(q), len(k)
    i, j = torch.arange(tq, device="cuda")[:, None] + tk - tq, torch.arange(tk, device="cuda")[None, :]
    s = (q @ k.T) * scale
    derivative = torch.ones_like(s)
    if cap:
        derivative = torch.cosh(s / cap) ** -2
        s = cap * torch.tanh(s / cap)
    if slope is not None:
        s = s - slope * (i - j).abs()
    hidden = torch.zeros(tq, tk, dtype=torch.bool, device="cuda")
    if span is not None:
        hidden |= (j < span[:, :1]) | (j >= span[:, 1:])
    if causal:
        hidden |= j > i
    s = torch.where(hidden, torch.full_like(s, -math.inf), s)
    if stat is None:
        stat = torch.logsumexp(s, 1)
    p = torch.exp(s - torch.where(stat == -math.inf, torch.zeros_like(stat), stat)[:, None])
    return p, stat, derivative


def _exact_attention(q, k, v, spans, slopes, scale, cap, causal, backward=None):
    """(out, statistics), or (dq, dk, dv) for ``backward`` = (out, statistics, do), which are inputs as the forward pass rounded them."""
    b, _, h, _ = q.shape
    group = h // k.shape[2]
    results = [torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)] if backward else [
        torch.zeros_like(q), torch.zeros(b, h, q.shape[1], dtype=torch.float64, device="cuda")]
    for n in range(b):
        span = None if spans is None else spans[n]
        for head in range(h):
            shared = head // group
            a, c, w = q[n, :, head], k[n, :, shared], v[n, :, shared]
            slope = None if slopes is None else slopes[head]
            if backward is None:
                p, results[1][n, head], _ = _exact_probabilities(a, c, span, slope, scale, cap, causal)
                results[0][n, :, head] = p @ w
            else:
                out, stat, do = backward
                p, _, derivative = _exact_probabilities(a, c, span, slope, scale, cap, causal, stat[n, head])
                d = do[n, :, head]
                ds = p * (d @ w.T - (d * out[n, :, head]).sum(1, keepdim=True)) * derivative * scale
                results[0][n, :, head] = ds @ c
                results[1][n, :, shared] += ds.T @ a
                results[2][n, :, shared] += p.T @ d
    return results


def exact(case, seed):
    """The definitions in 64 bits."""
    t = {name: v.double() for name, v in _inputs(case, seed).items()}
    kind, h, hk, d = case["kind"], case["heads"], case["key_heads"], case["dim"]
    if kind == "heads":
        turn = t["positions"], t["frequencies"], case["interleaved"], AMPLITUDE
        if case["direction"] == "backward":
            found = {}
            for x, g, dy, heads in (("q", "gq", "dq", h), ("k", "gk", "dk", hk)):
                leaves = t[x].requires_grad_(), t[g].requires_grad_()
                found["d%s_in" % x], found["d" + g] = torch.autograd.grad(_exact_heads(*leaves, heads, *turn), leaves, t[dy])
            return {name: found[name] for name in ("dq_in", "dk_in", "dgq", "dgk")}
        q, k = _exact_heads(t["q"], t["gq"], h, *turn), _exact_heads(t["k"], t["gk"], hk, *turn)
        if case["direction"] == "forward":
            return {"q_out": q, "k_out": k}
        for row, slot in enumerate(t["slots"][0].tolist()):
            t["k_cache"][0, int(slot)] = k[row]
            t["v_cache"][0, int(slot)] = t["v"][row]
        return {"q_out": q, "k_cache": t["k_cache"], "v_cache": t["v_cache"]}
    causal = kind != "cache" and case["mask"] == "causal"
    if kind != "sublayer":
        backward = (t["out"], t["stat"], t["do"]) if "do" in t else None
        found = _exact_attention(t["q"], t["k"], t["v"], t.get("spans"), t.get("slopes"), _scale(case), case["cap"], causal, backward)
        if backward:
            return dict(zip(("dq", "dk", "dv"), found))
        return dict(zip(("out", "stat"), found)) if kind == "attention" and case["direction"] == "train" else {"out": found[0]}
    # the sublayer's gradients by differentiating the definition up to the heads' attention and behind it
    b, n = case["batch"], case["tokens"]
    names = ("x", "gamma", "beta", "wq", "wk", "wv", "gq", "gk")
    leaves = [t[name].requires_grad_() for name in names]
    x = t["x"]
    centred = x - x.sum(1, keepdim=True) / x.shape[1]
    norm = centred / ((centred ** 2).sum(1, keepdim=True) / x.shape[1] + NORM_EPS) ** 0.5 * t["gamma"] + t["beta"]
    turn = t["positions"], t["frequencies"], False, 1.0
    q = _exact_heads(norm @ t["wq"], t["gq"], h, *turn).reshape(b, n, h, d)
    k = _exact_heads(norm @ t["wk"], t["gk"], hk, *turn).reshape(b, n, hk, d)
    v = (norm @ t["wv"]).reshape(b, n, hk, d)
    values = q.detach(), k.detach(), v.detach()
    shared = t.get("spans"), None, _scale(case), 0.0, causal
    out, stat = _exact_attention(*values, *shared)
    att = out.reshape(b * n, h * d)
    do = (t["dy"] @ t["wo"].T).reshape(b, n, h, d)
    inner = _exact_attention(*values, *shared, (out, stat, do))
    found = torch.autograd.grad((q, k, v), leaves, inner)
    grads = {"d" + name: g for name, g in zip(names, found)}
    grads["dx"] = grads["dx"] + t["dy"]
    grads.update(y=(x + att @ t["wo"]).detach(), dwo=att.T @ t["dy"])
    return {name: grads[name] for name in ("y", "dx", "dgamma", "dbeta", "dwq", "dwk", "dwv", "dwo", "dgq", "dgk")}


# ---------------------------------------------------------------------- what it has to cost

def work(case):
    """Each input read once and each output written once; of a cache what the sequences have used; the products'
    multiply-adds over the pairs that are seen, and a handful of operations an element elsewhere."""
    kind, h, hk, d = case["kind"], case["heads"], case["key_heads"], case["dim"]
    if kind == "heads":
        n = case["rows"] * (h + hk) * d
        if case["direction"] == "backward":
            return {"bytes": 4 * (3 * n + 4 * d + case["rows"]), "flops": 20 * n}
        moved = 2 * n + 2 * d + case["rows"] + (2 * case["rows"] * hk * d if case["direction"] == "serve" else 0)
        return {"bytes": 4 * moved, "flops": 8 * n}
    products = 2 * h * d * _pairs(case)   # of one product of queries and keys
    if kind == "cache":
        tokens = case["batch"] * case["queries"]
        return {"bytes": 4 * (2 * tokens * h * d + 2 * sum(_lengths(case)) * hk * d), "flops": 2 * products}
    tokens = case["batch"] * case["tokens"]
    if kind == "attention":
        if case["direction"] == "backward":
            return {"bytes": 4 * tokens * (4 * h * d + 4 * hk * d + h), "flops": 5 * products}
        return {"bytes": 4 * tokens * (2 * h * d + 2 * hk * d + (h if case["direction"] == "train" else 0)), "flops": 2 * products}
    # between the two passes the projections, their rotated forms, the attention's output and its statistics are kept
    w = case["width"]
    weights = 2 * w * (h + hk) * d
    return {"bytes": 4 * (4 * tokens * w + 2 * weights + 2 * tokens * (3 * h + 3 * hk) * d),
            "flops": 6 * tokens * weights + 7 * products}
