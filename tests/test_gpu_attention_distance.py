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
