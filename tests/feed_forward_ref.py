"""The operators of a feed-forward sublayer in float64, and how far an fp32 evaluation may be from them.

Every bound is first-order: u = 2^-24 is the largest relative error of one fp32 rounding, a sum whose longest chain of
additions has n members is off by at most n u times the sum of its members' magnitudes, and an error in an operand is
carried through the derivative.  Chains of the kernels: layer norm adds at most 16 values in a lane, 6 steps across a wave and 16 waves
(38), or a row's columns / 1024 in a lane where registers do not hold it.
"""
import math

import numpy as np

U = 2.0 ** -24


def _rows(x, cols):
    return np.asarray(x, np.float64).reshape(-1, cols)


def norm_chain(cols):
    return 40 + cols / 1024


class Norm(object):
    """Layer norm of x over its last axis and its gradients, with their bounds."""

    def __init__(self, x, gamma, beta, eps):
        self.shape, cols = x.shape, x.shape[-1]
        x = _rows(x, cols)
        self.gamma, self.beta = np.asarray(gamma, np.float64), np.asarray(beta, np.float64)
        mean = x.mean(1, keepdims=True)
        self.s = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
        self.xh = (x - mean) * self.s
        self.y = (self.gamma * self.xh + self.beta).reshape(self.shape)
        # xh: the mean is off by n u mean|x|, everything else by a few roundings and half the variance's n u
        n = norm_chain(cols)
        self.d_xh = U * n * (np.abs(x).mean(1, keepdims=True) * self.s + np.abs(self.xh) + 8 * U)
        self.y_tol = (np.abs(self.gamma) * (self.d_xh + 4 * U * np.abs(self.xh))
                      + 2 * U * (np.abs(self.beta) + np.abs(self.y.reshape(x.shape)))).reshape(self.shape)
        self.n = n

    def backward(self, dy):
        """dx, dgamma, dbeta and their bounds."""
        dy = _rows(dy, self.shape[-1])
        a = dy * self.gamma
        m1, m2 = a.mean(1, keepdims=True), (a * self.xh).mean(1, keepdims=True)
        dx = self.s * (a - m1 - self.xh * m2)
        # the two means are off by n u of their members and by what xh is off; so is the product with xh
        d_m1 = U * (self.n + 2) * np.abs(a).mean(1, keepdims=True)
        d_m2 = (U * (self.n + 4) * np.abs(a * self.xh).mean(1, keepdims=True)
                + (np.abs(a) * self.d_xh).mean(1, keepdims=True))
        inner = np.abs(a) + np.abs(m1) + np.abs(self.xh * m2)
        dx_tol = self.s * (d_m1 + np.abs(self.xh) * d_m2 + self.d_xh * np.abs(m2) + U * (self.n + 8) * inner)
        rows = len(dy)
        chain = 64 + rows / 16   # rows of one workgroup, its four rows, every 32nd piece, 32 of those
        dgamma, dbeta = (dy * self.xh).sum(0), dy.sum(0)
        dgamma_tol = (U * chain * np.abs(dy * self.xh) + np.abs(dy) * self.d_xh).sum(0)
        dbeta_tol = (U * chain * np.abs(dy)).sum(0)
        return [(dx.reshape(self.shape), dx_tol.reshape(self.shape)), (dgamma, dgamma_tol), (dbeta, dbeta_tol)]


def product(a, b, d_a=0.0, d_b=0.0):
    """a b and its bound.  The engines add at least eight products at a time; two or three slices of an operand leave off at
    most 2 u of it, and where slices are scaled by their row's largest value 2^-40 of that."""
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    k = a.shape[1]
    if a.size == 0 or b.size == 0:
        return a @ b, np.zeros((a.shape[0], b.shape[1]))
    A, B = np.abs(a), np.abs(b)
    scaled = 2.0 ** -40 * (A.max(1, keepdims=True) * B.sum(0) + A.sum(1, keepdims=True) * B.max(0))
    tol = U * (k / 8 + 16) * (A @ B) + scaled
    if np.ndim(d_a):
        tol = tol + d_a @ B
    if np.ndim(d_b):
        tol = tol + A @ d_b
    return a @ b, tol


_erf = np.vectorize(math.erf, otypes=[np.float64])


def act_and_slope(g, activation):
    """act(g), act'(g) and a bound of |act''|."""
    if activation == "relu":
        return np.maximum(g, 0), (g > 0).astype(np.float64), 0.0
    if activation == "gelu":
        cdf = 0.5 * (1 + _erf(g / math.sqrt(2)))
        pdf = np.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
        return g * cdf, cdf + g * pdf, 0.8
    s = 1 / (1 + np.exp(-g))
    if activation == "sigmoid":
        return s, s * (1 - s), 0.1
    return g * s, s * (1 + g * (1 - s)), 0.5


def gated(x, gate, up, activation):
    """(pre, its bound), (h, its bound)"""
    g, d_g = product(x, gate)
    u, d_u = product(x, up)
    act, slope, _ = act_and_slope(g, activation)
    h = act * u
    # act itself: a few roundings of |g| or of 1
    d_act = 8 * U * (np.abs(g) if activation in ("gelu", "silu", "relu") else 1.0)
    if activation == "relu":   # on the other side of zero where g is rounding
        d_act = np.where(np.abs(g) <= d_g, d_g, d_act)
    h_tol = np.abs(u) * (np.abs(slope) * d_g + d_act + d_g * d_g) + np.abs(act) * d_u + d_g * d_u + 4 * U * np.abs(h)
    return (np.stack([g, u]), np.stack([d_g, d_u])), (h, h_tol)


def pointwise_gradient(pre, dh, activation):
    """(dg, du) and their bounds for given projections"""
    g, u, dh = (np.asarray(v, np.float64) for v in (pre[0], pre[1], dh))
    act, slope, _ = act_and_slope(g, activation)
    d_act = 8 * U * (np.abs(g) if activation != "sigmoid" else 1.0)
    # the slope is a sum of terms of at most 1 + |g|, each a few roundings of exp and of a reciprocal off
    d_slope = 0.0 if activation == "relu" else 16 * U * (1 + np.abs(g))
    dg, du = dh * u * slope, dh * act
    return (np.stack([dg, du]),
            np.stack([np.abs(dh * u) * (d_slope + 4 * U * np.abs(slope)), np.abs(dh) * (d_act + 4 * U * np.abs(act))]))


def gated_backward(x, gate, up, dpre, d_dpre):
    """dx, dgate, dup and their bounds from the projections' gradients"""
    both = np.concatenate([dpre[0], dpre[1]], 1)
    d_both = np.concatenate([d_dpre[0], d_dpre[1]], 1)
    weights = np.concatenate([np.asarray(gate, np.float64), np.asarray(up, np.float64)], 1)
    xt = np.asarray(x, np.float64).T
    return [product(both, weights.T, d_a=d_both), product(xt, dpre[0], d_b=d_dpre[0]), product(xt, dpre[1], d_b=d_dpre[1])]


def philox(count, seed, offset, first=0):
    """The generator's words, one an element, from element ``first`` on, a multiple of four."""
    low = np.uint64(0xFFFFFFFF)
    block = np.arange(first // 4, first // 4 + (count + 3) // 4, dtype=np.uint64)
    c = [block & low, block >> np.uint64(32), np.full_like(block, offset & 0xFFFFFFFF), np.full_like(block, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p, q = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(q >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), q & low, (p >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return np.stack(c, 1).ravel()[:count]


def kept(count, dropout, seed, offset, first=0):
    return philox(count, seed, offset, first) >= np.uint64(math.floor(float(np.float32(dropout)) * 2 ** 32))


def assert_within(got, ref, tol, what):
    got = np.asarray(got, np.float64)
    assert got.shape == ref.shape, "%s: shape %s, not %s" % (what, got.shape, ref.shape)
    off = np.abs(got - ref) - tol
    bad = ~(off <= 0)
    assert not bad.any(), "%s: %d of %d values are out of bounds; the worst is off by %.3g where %.3g is allowed" % (
        what, bad.sum(), bad.size, np.abs(got - ref).ravel()[np.nanargmax(np.where(bad, np.abs(off), -1))],
        np.broadcast_to(tol, ref.shape).ravel()[np.nanargmax(np.where(bad, np.abs(off), -1))])
