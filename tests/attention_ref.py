"""The operators of an attention sublayer in float64, and how far an fp32 evaluation may be from them.

Every bound is first-order: u = 2^-24 is the largest relative error of one fp32 rounding, a sum whose longest chain of
additions has n members is off by at most n u times the sum of its members' magnitudes, and an error in an operand is
carried through the derivative.  A product's operands may be split into pairs of fp16 numbers that leave off 4 u of a product, or
2^-38 of the largest values of their tiles: `floor`.
"""
import numpy as np

U = 2.0 ** -24
FLOOR = 2.0 ** -38


class Heads(object):
    """Norm and rotation of x [rows, heads, dim]; gamma, frequencies may be None."""

    def __init__(self, x, gamma, positions, frequencies, amplitude, interleaved, eps):
        x = np.asarray(x, np.float64)
        self.gamma = None if gamma is None else np.asarray(gamma, np.float64)
        rows, _, dim = x.shape
        if gamma is not None:
            self.s = 1 / np.sqrt((x * x).mean(2, keepdims=True) + np.float64(np.float32(eps)))
            self.n = x * self.s
            y = self.n * self.gamma
        else:
            y = x
        self.turn = None
        if frequencies is not None:
            f = np.asarray(frequencies, np.float64)
            p = np.asarray(positions, np.float64).reshape(-1)
            angle = np.tile(p, rows // max(len(p), 1))[:, None, None] * f
            self.turn = (np.cos(angle), np.sin(angle), float(np.float32(amplitude)), interleaved)
        # the norm: sums of dim squares in chains of at most 24, a root, a division, two products: 16 u; the turn: two
        # products, a sum, sine and cosine a few u off each: 8 u of both columns
        self.y = self._rotate(y, 1)
        near = self._rotate_abs(np.abs(y))
        self.y_tol = 32 * U * near

    def _columns(self, dim):
        half = self.turn[0].shape[2]
        first = np.arange(0, 2 * half, 2) if self.turn[3] else np.arange(half)
        return first, first + (1 if self.turn[3] else half)

    def _rotate(self, y, sign):
        if self.turn is None:
            return y
        c, s, amp, _ = self.turn
        a, b = self._columns(y.shape[2])
        out = y.copy()
        out[..., a] = amp * (y[..., a] * c - sign * y[..., b] * s)
        out[..., b] = amp * (sign * y[..., a] * s + y[..., b] * c)
        return out

    def _rotate_abs(self, y):
        if self.turn is None:
            return y
        a, b = self._columns(y.shape[2])
        out = y.copy()
        out[..., a] = out[..., b] = self.turn[2] * (y[..., a] + y[..., b])
        return out

    def backward(self, dy):
        """dx, dgamma (None without a norm) and their bounds."""
        dy = np.asarray(dy, np.float64)
        da, d_da = self._rotate(dy, -1), 16 * U * self._rotate_abs(np.abs(dy))
        if self.gamma is None:
            return (da, d_da), None
        t = da * self.gamma
        c = (t * self.n).mean(2, keepdims=True)
        dx = self.s * (t - self.n * c)
        d_t = d_da * np.abs(self.gamma) + U * np.abs(t)
        d_c = (d_t * np.abs(self.n) + 24 * U * np.abs(t * self.n)).mean(2, keepdims=True)
        dx_tol = self.s * (d_t + np.abs(self.n) * d_c + 24 * U * (np.abs(t) + np.abs(self.n * c)))
        dgamma = (da * self.n).sum((0, 1))
        chain = 96 + da.shape[0] * da.shape[1] / 64   # a lane's rows, a workgroup's groups, 32 pieces
        dgamma_tol = ((chain + 24) * U * np.abs(da * self.n) + d_da * np.abs(self.n)).sum((0, 1))
        return (dx, dx_tol), (dgamma, dgamma_tol)


def seen(batch, tq, tk, spans, causal):
    """[batch, queries, keys]"""
    j = np.arange(tk)
    mask = np.ones((batch, tq, tk), bool)
    if spans is not None:
        s = np.broadcast_to(np.asarray(spans, np.float64).reshape(-1, tq, 2), (batch, tq, 2))
        mask &= (j >= s[..., :1]) & (j < s[..., 1:])
    if causal:
        mask &= j <= np.arange(tq)[:, None] + tk - tq
    return mask


def _largest(x):
    x = np.abs(x[np.isfinite(x)])
    return x.max() if x.size else 0.0


class Attention(object):
    """q [batch, queries, heads, dim], k and v [batch, keys, key heads, dim].  What a query does not see must be finite here."""

    def __init__(self, q, k, v, spans=None, slopes=None, scale=1.0, cap=0.0, causal=False):
        self.q, self.k, self.v = (np.asarray(x, np.float64) for x in (q, k, v))
        b, tq, h, d = self.q.shape
        tk, hk = self.k.shape[1:3]
        self.group = h // hk
        self.scale, self.cap = float(np.float32(scale)), float(np.float32(cap))
        self.mask = seen(b, tq, tk, spans, causal)[:, None]
        k_all, v_all = self._shared(self.k), self._shared(self.v)
        qh = self.q.transpose(0, 2, 1, 3)
        s = self.scale * (qh @ k_all.transpose(0, 1, 3, 2))
        size = self.scale * (np.abs(qh) @ np.abs(k_all).transpose(0, 1, 3, 2))
        e = U * (d / 8 + 24) * size + FLOOR * self.scale * d * _largest(self.q) * _largest(self.k)
        self.slope = np.ones_like(s)
        self.e_slope = np.zeros_like(s)
        if self.cap:
            t = np.tanh(s / self.cap)
            self.slope = 1 - t * t
            self.e_slope = 2 * np.abs(t) * e / self.cap + 12 * U
            e = e * self.slope + 6 * U * self.cap * np.abs(t) + e * e / self.cap
            s = self.cap * t
        if slopes is not None:
            ahead = np.abs(np.arange(tq)[:, None] + tk - tq - np.arange(tk))
            bias = np.asarray(slopes, np.float64)[:, None, None] * ahead
            s = s - bias
            e = e + 3 * U * bias
        self.e = e + 4 * U * np.abs(s)
        self.s = np.where(self.mask, s, -np.inf)
        top = self.s.max(3, initial=-np.inf, keepdims=True) if tk else np.full(s.shape[:3] + (1,), -np.inf)
        top = np.where(np.isfinite(top), top, 0)
        p = np.exp(self.s - top)
        total = p.sum(3, keepdims=True)
        some = total > 0
        with np.errstate(divide="ignore"):
            self.stat = np.where(some, top + np.log(total), -np.inf)[..., 0]
        self.p = p / np.where(some, total, 1)
        chain = tk / 2 + 64
        # where the exponents' differences are large, p is small
        e_p = self.e + 4 * U * (1 + np.abs(np.where(self.mask, self.s - top, 0)))
        mean = (self.p * e_p).sum(3, keepdims=True)
        self.out = (self.p @ v_all).transpose(0, 2, 1, 3)
        near = np.abs(v_all)
        out_tol = (self.p * (e_p + mean)) @ near + U * chain * (self.p @ near) + FLOOR * _largest(v_all) * some
        self.out_tol = 1.01 * out_tol.transpose(0, 2, 1, 3)
        self.stat_tol = 1.01 * (mean[..., 0] + U * (chain + 8) + 4 * U * np.where(np.isfinite(self.stat), np.abs(self.stat), 0))

    def _shared(self, x):
        """[batch, heads, keys, dim]"""
        return np.repeat(x.transpose(0, 2, 1, 3), self.group, 1)

    def _sum_group(self, x):
        b, h, n, d = x.shape
        return x.reshape(b, h // self.group, self.group, n, d).sum(2).transpose(0, 2, 1, 3)

    def backward(self, out, stat, do):
        """[(dq, bound), (dk, bound), (dv, bound)] from the forward pass's fp32 results."""
        out, stat, do = (np.asarray(x, np.float64) for x in (out, stat, do))
        d, tk, tq = self.q.shape[3], self.k.shape[1], self.q.shape[1]
        qh, dh, oh = (x.transpose(0, 2, 1, 3) for x in (self.q, do, out))
        k_all, v_all = self._shared(self.k), self._shared(self.v)
        at = np.where(np.isfinite(stat), stat, 0)[..., None]
        p = np.exp(self.s - at)
        e_p = self.e + 4 * U * (1 + np.abs(at))
        dp = dh @ v_all.transpose(0, 1, 3, 2)
        e_dp = (U * (d / 8 + 24) * (np.abs(dh) @ np.abs(v_all).transpose(0, 1, 3, 2)) + FLOOR * d * _largest(do) * _largest(self.v))
        delta = (dh * oh).sum(3, keepdims=True)
        e_delta = U * (d / 64 + 12) * np.abs(dh * oh).sum(3, keepdims=True)
        diff = dp - delta
        ds = p * diff * self.slope
        e_ds = p * ((e_dp + e_delta + np.abs(diff) * (e_p + 6 * U)) * self.slope + np.abs(diff) * self.e_slope)
        # what a split of p or ds leaves off: of its bound, which no value passes
        f_p = FLOOR * np.ones_like(p) * self.mask
        f_ds = FLOOR * d * _largest(do) * _largest(self.v) * np.ones_like(p) * self.mask
        near = [np.abs(x) for x in (qh, k_all, dh)]
        of = [_largest(x) for x in (self.q, self.k, do)]

        def product(w, e_w, x, near_x, n, largest, floor_w):
            tol = (e_w + floor_w) @ near_x + U * (n / 2 + 64) * (np.abs(w) @ near_x) + FLOOR * largest * np.abs(w).sum(3, keepdims=True)
            return w @ x, tol

        def turned(x):
            return x.transpose(0, 1, 3, 2)
        rows = tq * self.group
        dq, dq_tol = product(ds, e_ds, k_all, near[1], tk, of[1], f_ds)
        dk, dk_tol = product(turned(ds), turned(e_ds), qh, near[0], rows, of[0], turned(f_ds))
        dv, dv_tol = product(turned(p), turned(p * e_p), dh, near[2], rows, of[2], turned(f_p))
        return [(self.scale * dq.transpose(0, 2, 1, 3), 1.01 * self.scale * dq_tol.transpose(0, 2, 1, 3)),
                (self.scale * self._sum_group(dk), 1.01 * self.scale * self._sum_group(dk_tol)),
                (self._sum_group(dv), 1.01 * self._sum_group(dv_tol))]


def assert_within(got, ref, tol, what):
    got = np.asarray(got, np.float64)
    assert got.shape == ref.shape, "%s: shape %s, not %s" % (what, got.shape, ref.shape)
    tol = np.broadcast_to(tol, ref.shape)
    same = (got == ref) | (np.isnan(got) & np.isnan(ref))
    with np.errstate(invalid="ignore"):
        bad = ~(same | (np.abs(got - ref) <= tol))
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, np.nan_to_num(np.abs(got - ref) / np.maximum(tol, 1e-300), nan=np.inf), 0)), ref.shape)
        raise AssertionError("%s: %d of %d values are out of bounds; at %s %.9g for %.9g, %.3g allowed"
                             % (what, bad.sum(), bad.size, at, got[at], ref[at], tol[at]))
