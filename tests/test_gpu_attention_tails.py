"""Attention of few queries over caches that fill their memory: heads whose length is no multiple of four, up to the last key of the last head."""
import numpy as np
import pytest

import attention_ref as ref
from parity import stable_seed
from test_gpu_attention import _check, _data

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("b,tq,tk,h,hk,d", [(1, 1, 4096, 4, 4, 66), (1, 2, 8192, 2, 1, 66), (1, 1, 1, 1, 1, 1), (2, 3, 64, 2, 2, 2), (2, 1, 128, 3, 1, 1),
                                            (1, 4, 512, 1, 1, 129), (1, 1, 256, 2, 2, 254), (1, 20, 256, 1, 1, 127)])
def test_to_the_last_key(rt, b, tq, tk, h, hk, d):
    """The last keys' largest scores make them count; what a head's last columns hold is seen in the output."""
    q, k, v, do = _data(b, tq, tk, h, hk, d, stable_seed((tk, d)))
    k[:, -1] *= 2
    out, stat, _ = _check(rt, q, k, v, do, causal=True, backward=False)
    spans = np.zeros((tq, 2), np.float32)
    spans[:, 0], spans[:, 1] = tk - 1, tk   # the last key alone: its value comes out
    out, _, _ = _check(rt, q, k, v, do, spans=spans, backward=False)
    np.testing.assert_array_equal(out, np.repeat(v[:, -1:], h // hk, 2).repeat(tq, 1))
