"""The distance term over a cache whose end is not used."""
import numpy as np
import pytest

import attention_ref as ref
from test_gpu_attention import _check, _data, _device, _empty, _run

pytestmark = pytest.mark.gpu


def _cache(rt_seed, b, tq, capacity, used, h, hk, d):
    q, k, v, do = _data(b, tq, capacity, h, hk, d, rt_seed)
    k[:, used:] = v[:, used:] = np.nan
    return q, k, v, do, 2.0 ** -np.arange(1, h + 1)


# few rows alone and cut, tiles of the fp32 instruction (longer heads) and of pairs, cut along the keys and not
@pytest.mark.parametrize("tq,capacity,used,h,hk,d", [(1, 131072, 1000, 4, 2, 64), (5, 16384, 1000, 8, 8, 64), (5, 1500, 1237, 8, 8, 64),
                                                     (40, 131072, 1000, 4, 2, 64), (70, 20000, 900, 2, 2, 200), (600, 30000, 600, 2, 1, 64),
                                                     (20, 65536, 50, 1, 1, 128)])
def test_shares_do_not_depend_on_the_capacity(rt, tq, capacity, used, h, hk, d):
    """Where queries see earlier keys alone, every score moves by the same amount: the outputs are those of the used part alone, and the statistics
    differ by slope * (capacity - used)."""
    from tinyflow_amd import gpu_op
    q, k, v, _, slopes = _cache(5, 1, tq, capacity, used, h, hk, d)
    spans = gpu_op.attention_spans(tq, capacity, causal=True, used=[used])
    out, stat, _ = _run(rt, q, k, v, None, spans=spans, slopes=slopes, backward=False)
    want = ref.Attention(q, k[:, :used], v[:, :used], None, slopes, d ** -0.5, causal=True)
    ref.assert_within(out, want.out, want.out_tol, "out")
    moved = want.stat - (slopes * (capacity - used))[:, None]
    ref.assert_within(stat, moved, want.stat_tol + ref.U * np.abs(moved), "statistics")


@pytest.mark.parametrize("cap", [0.0, 10.0])
@pytest.mark.parametrize("tq,capacity,used,h,hk,d", [(5, 4000, [900, 4000], 4, 2, 64), (40, 3000, [700, 40], 4, 2, 64), (200, 1500, [1237, 200], 2, 2, 96),
                                                     (150, 131072, [151, 1000], 2, 1, 24), (33, 600, [400, 33], 1, 1, 160)])
def test_queries_at_their_own_places(rt, tq, capacity, used, h, hk, d, cap):
    """A prefix that is seen in both directions, over caches that are not full: keys in front of a query and behind it count by their distance
    from it, forward and backward, as in the used part alone."""
    from tinyflow_amd import gpu_op
    b = len(used)
    q, k, v, do = _data(b, tq, capacity, h, hk, d, 6)
    slopes = 2.0 ** -np.arange(1, h + 1)
    prefix = [n - tq // 2 for n in used]
    spans = gpu_op.attention_spans(tq, capacity, causal=True, used=used, prefix=prefix, positions=True)
    assert spans.shape == (b, tq, 3)
    for n in range(b):
        k[n, used[n]:] = v[n, used[n]:] = np.nan
    out, stat, grads = _run(rt, q, k, v, do, spans=spans, slopes=slopes, cap=cap)
    for n in range(b):
        own = slice(n, n + 1), slice(0, used[n])
        alone = gpu_op.attention_spans(tq, used[n], causal=True, prefix=[prefix[n]])
        want = ref.Attention(q[own[:1]], k[own], v[own], alone, slopes, d ** -0.5, cap)
        ref.assert_within(out[own[:1]], want.out, want.out_tol, "out of %d" % n)
        ref.assert_within(stat[own[:1]], want.stat, want.stat_tol, "statistics of %d" % n)
        values = want.backward(out[own[:1]], stat[own[:1]], do[own[:1]])
        for what, got, (value, tol) in zip(("dq", "dk", "dv"), (grads[0][own[:1]], grads[1][own], grads[2][own]), values):
            ref.assert_within(got, value, tol, "%s of %d" % (what, n))
        assert not grads[1][n, used[n]:].any() and not grads[2][n, used[n]:].any()


@pytest.mark.parametrize("tq", [3, 70])
def test_causal_from_the_given_places(rt, tq):
    """``causal`` asks for the key that a query stands at, whichever that is, in any order; far outside of the keys it sees none or all."""
    rng = np.random.RandomState(7)
    tk = 200
    at = rng.permutation(tk)[:tq].astype(np.float32)
    at[0], at[1] = -1e9, 1e9
    spans = np.stack([np.zeros(tq), np.full(tq, tk), at], 1).astype(np.float32)
    q, k, v, do = _data(2, tq, tk, 2, 1, 40, 8)
    out, stat, grads = _run(rt, q, k, v, do, spans=spans, causal=True)
    seen = np.stack([np.zeros(tq), np.minimum(at + 1, tk)], 1).astype(np.float32)
    want = ref.Attention(q, k, v, seen, None, 40 ** -0.5)
    ref.assert_within(out, want.out, want.out_tol, "out")
    ref.assert_within(stat, want.stat, want.stat_tol, "statistics")
    for what, got, (value, tol) in zip(("dq", "dk", "dv"), grads, want.backward(out, stat, do)):
        ref.assert_within(got, value, tol, what)
