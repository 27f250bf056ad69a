"""The backward pass where a key or a value is not finite: gradients of what cannot see it have their numbers, and those of what does are not finite,
in whatever tile they are."""
import numpy as np
import pytest

import attention_ref as ref
from test_gpu_attention import _data, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("which", ["key", "value"])
@pytest.mark.parametrize("d", [64, 128])
def test_documents_keep_it_to_themselves(rt, monkeypatch, split, bad, which, d):
    """Two documents, the border inside of a block of 32 rows; the bad number lies two tiles of keys in front of it."""
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    q, k, v, do = _data(1, 400, 400, 2, 1, d, 21)
    border = 144
    spans = np.zeros((400, 2), np.float32)
    spans[:border, 1] = border
    spans[border:] = border, 400
    own = slice(border, 400)
    want = ref.Attention(q[:, own], k[:, own], v[:, own], None, None, d ** -0.5)
    (k if which == "key" else v)[0, 5, 0, 3] = bad
    out, stat, grads = _run(rt, q, k, v, do, spans=spans)
    ref.assert_within(out[:, own], want.out, want.out_tol, "out")
    ref.assert_within(stat[..., own], want.stat, want.stat_tol, "statistics")
    for what, got, (value, tol) in zip(("dq", "dk", "dv"), grads, want.backward(out[:, own], stat[..., own], do[:, own])):
        ref.assert_within(got[:, own], value, tol, what)
    # The first document's rows all see it; an infinite key's score may be -infinity, and its share 0.
    if which == "key" and bad == np.inf:
        return
    assert not np.isfinite(grads[0][:, :border]).all(3).any()
    assert not np.isfinite(grads[1][:, :border]).all(3).any()


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("d", [64, 128])
def test_no_gradient_becomes_zero(rt, monkeypatch, split, d):
    """Causal rows from the fifth on see a NaN: every key's gradient has one, also where the tile of keys holds only finite numbers."""
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    q, k, v, do = _data(1, 400, 400, 2, 1, d, 22)
    clean = v.copy()
    v[0, 5, 0, 3] = np.nan
    _, _, (dq, dk, dv) = _run(rt, q, k, v, do, causal=True)
    assert np.isnan(dk).all() and np.isnan(dq[:, 5:]).all() and np.isfinite(dv).all() and np.isfinite(dq[:, :5]).all()
    k[0, 5, 0, 3] = np.nan
    _, _, (dq, dk, dv) = _run(rt, q, k, clean, do, causal=True)
    assert np.isnan(dk).all() and np.isnan(dv).all() and np.isnan(dq[:, 5:]).any(3).all() and np.isfinite(dq[:, :5]).all()


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("d", [64, 128])
def test_shares_past_the_largest_number(rt, monkeypatch, split, d):
    """Statistics far below the scores' make every share infinite: so are the gradients, not 0."""
    from tinyflow_amd import gpu_op
    from test_gpu_attention import _device, _empty
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    q, k, v, do = _data(1, 300, 300, 2, 1, d, 23)
    out, stat, _ = _run(rt, q, k, v, do, backward=False)
    grads = [_empty(rt, x.shape) for x in (q, k, v)]
    a = _device(rt, q, k, v) + [None, None] + _device(rt, out, stat - 300, do)
    assert gpu_op.attention_backward(*a, *grads, 1, 2, 1, d ** -0.5, 0.0, False, rt.stream) == 0
    for g in grads:
        assert not np.isfinite(g.asnumpy()).any()
