"""Attention on fp16 pairs where splitting could go wrong: blocks of unlike magnitude, of zeros, of rows too unlike for one exponent, and what is not
finite; both engines against float64."""
import numpy as np
import pytest

import attention_ref as ref
from parity import stable_seed
from test_gpu_attention import _check, _data, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("d", [24, 64, 96, 128])
def test_both_engines(rt, monkeypatch, split, d):
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    _check(rt, *_data(2, 333, 290, 4, 2, d, d), causal=True)
    _check(rt, *_data(1, 200, 700, 2, 1, d, d), slopes=np.array([0.5, 0.01]), cap=8.0)


def test_the_engines_are_two(rt, monkeypatch):
    """TINYFLOW_SPLIT=0 reaches the calls: the bits differ."""
    outs = []
    for split in ("0", "1"):
        monkeypatch.setenv("TINYFLOW_SPLIT", split)
        outs.append(_run(rt, *_data(1, 600, 600, 4, 2, 64, 3), causal=True))
    assert (outs[0][0] != outs[1][0]).any() and (outs[0][2][0] != outs[1][2][0]).any()


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("power", [-30, -8, 8, 25])
def test_blocks_of_unlike_magnitude(rt, which, power):
    """Every other block of 32 rows of one operand by a power of two: sums change their unit on the way, up and down.  (Bounds are of the call's
    largest values, so the small blocks are compared by themselves below.)"""
    a = _data(2, 300, 300, 2, 1, 64, 4)
    x = a[which].reshape(2, 300, -1)
    blocks = np.arange(300) // 32 % 2 == 1
    x[:, blocks] *= np.float32(2.0 ** (power if which > 1 else np.clip(power, -8, 3)))   # scores stay in the exponential's range
    _check(rt, *a, causal=True)


def test_small_blocks_by_themselves(rt):
    """Gradients of documents that are 2^-40 of their neighbours': each document's results have their own digits."""
    from tinyflow_amd import gpu_op
    q, k, v, do = _data(1, 320, 320, 2, 2, 64, 5)
    documents = np.arange(320) // 80
    small = documents % 2 == 1
    do[:, small] *= np.float32(2.0 ** -40)
    v[:, small] *= np.float32(2.0 ** -20)
    spans = gpu_op.attention_spans(320, documents=documents, causal=True)
    out, stat, grads = _run(rt, q, k, v, do, spans=spans)
    for n in range(4):
        own = documents == n
        want = ref.Attention(q[:, own], k[:, own], v[:, own], None, None, 0.125, causal=True)
        ref.assert_within(out[:, own], want.out, want.out_tol, "out of document %d" % n)
        values = want.backward(out[:, own], stat[:, :, own], do[:, own])
        for what, got, (value, tol) in zip(("dq", "dk", "dv"), grads, values):
            off = np.linalg.norm(got[:, own] - value) / np.linalg.norm(value)
            # a block of 32 rows that spans two documents is left to the fp32 kernels: sums of up to 80 rows or keys and 64 columns of products, each rounding
            # 2^-24 of a magnitude that cancellation makes up to four times the result's: 2^-24 (80 + 64) 4 < 2^-14.8
            assert off <= 2.0 ** -15, "%s of document %d is %.2g off" % (what, n, off)


@pytest.mark.parametrize("which", range(4))
def test_zeros(rt, which):
    a = _data(1, 160, 200, 2, 1, 40, 6)
    a[which][:, 30:130] = 0
    _check(rt, *a, causal=True)
    a[which][...] = 0
    _check(rt, *a, causal=True)


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e30])
def test_values_and_gradients_at_the_ends_of_the_range(rt, scale):
    """Values of 1e30 pass what a block may have and take the fp32 kernels; 1e-30 is held as it is."""
    q, k, v, do = _data(1, 150, 150, 2, 1, 32, 7)
    _check(rt, q, k, v * np.float32(scale), do / np.float32(max(scale, 1.0)), causal=True)


@pytest.mark.parametrize("which", [1, 2])
def test_rows_too_unlike_for_one_exponent(rt, which):
    """A key or value of 2^30 times its neighbours: its block is left to the fp32 kernels, in the tiles that see it."""
    a = _data(1, 400, 400, 2, 1, 64, 8)
    a[which][0, 210] *= np.float32(2.0 ** 30)
    if which == 1:
        a[0][0, :, :, :] *= np.float32(2.0 ** -26)   # scores stay in the exponential's range
    _check(rt, *a, causal=True)


@pytest.mark.parametrize("tq,tk", [(40, 3000), (128, 1100), (33, 257)])
def test_cut_along_the_keys(rt, tq, tk):
    """Few rows over many keys: pieces of their own units, joined."""
    q, k, v, do = _data(1, tq, tk, 2, 2, 48, 9)
    v[:, tk // 2:] *= np.float32(64)
    k[:, : tk // 3] *= np.float32(0.01)
    spans = np.zeros((tq, 2), np.float32)
    spans[:, 1] = tk - np.arange(tq)
    spans[::5] = 0
    _check(rt, q, k, v, do, spans=spans)


def test_one_bad_gradient_row(rt):
    """A gradient that is not finite reaches the keys that its query sees, and no others."""
    q, k, v, do = _data(1, 300, 300, 1, 1, 64, 10)
    out, stat, _ = clean = _run(rt, q, k, v, do, causal=True)
    do[0, 170, 0, 3] = np.inf
    dq, dk, dv = _run(rt, q, k, v, do, causal=True)[2]
    assert not np.isfinite(dv[0, :171, 0, 3]).any() and np.isfinite(dv[0, 171:]).all() and np.isfinite(dk[0, 171:]).all()
    assert np.isnan(dq[0, 170]).all() and np.isfinite(np.delete(dq[0], 170, 0)).all()
    for got, was in zip((dk, dv), clean[2][1:]):
        np.testing.assert_allclose(got[0, 171:], was[0, 171:], rtol=1e-4, atol=1e-6 * np.abs(was).max())


def test_more_rows_than_one_workgroup_a_cu(rt):
    """Tiles, pieces and heads beyond what is resident at once; the same bits again."""
    a = _data(3, 700, 700, 6, 3, 64, 11)
    first = _check(rt, *a, causal=True)
    again = _run(rt, *a, causal=True)
    np.testing.assert_array_equal(first[0], again[0])
    for x, y in zip(first[2], again[2]):
        np.testing.assert_array_equal(x, y)


@pytest.mark.parametrize("d", [64, 128])
def test_errors_of_rows_do_not_add_up(rt, d):
    """Of n independent errors with no mean the sum is beyond six times the root of their squares' sum once in 10^9.  What is summed here is what a gain
    of all queries, or of all keys, would have for its gradient."""
    q, k, v, do = _data(1, 1024, 1024, 8, 8, d, 12)
    out, stat, grads = _run(rt, q, k, v, do, causal=True)
    values = ref.Attention(q, k, v, None, None, 1 / np.sqrt(d), causal=True).backward(out, stat, do)
    for what, x, got, (want, _) in (("queries", q, grads[0], values[0]), ("keys", k, grads[1], values[1])):
        off = ((got - want) * x).sum(3)
        z = off.sum() / np.sqrt((off * off).sum())
        assert abs(z) <= 6, "the errors of the %s add up: %.1f" % (what, z)


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("tq,tk", [(1, 1200), (7, 2500), (40, 1500), (150, 1030)])
def test_gradients_of_few_queries(rt, monkeypatch, split, tq, tk):
    """The keys are cut; one key of another magnitude leaves its tile, all pieces of it, to the fp32 kernels."""
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    a = _data(2, tq, tk, 2, 2, 48, stable_seed((tq, tk)))
    _check(rt, *a, causal=True)
    a[2][1, 700] *= np.float32(2.0 ** 30)
    _check(rt, *a, causal=True)


def test_a_small_gradient_among_large_ones(rt):
    """Every 40th row's gradient is 2^-30 of the others': its dq has its own digits."""
    q, k, v, do = _data(1, 300, 300, 2, 1, 64, 13)
    rows = np.arange(300) % 40 == 7
    do[:, rows] *= np.float32(2.0 ** -30)
    out, stat, grads = _run(rt, q, k, v, do, causal=True)
    want = ref.Attention(q, k, v, None, None, 0.125, causal=True).backward(out, stat, do)[0][0]
    off = np.linalg.norm((grads[0] - want)[:, rows]) / np.linalg.norm(want[:, rows])
    # sums of up to 300 keys and 64 columns, each rounding 2^-24 of up to four times the result's magnitude: 2^-24 (300 + 64) 4 < 2^-13.4
    assert off <= 2.0 ** -13.4, "%.2g off" % off


@pytest.mark.parametrize("tq", [2048, 2049])
def test_spans_of_many_queries(rt, tq):
    """Keys in front of the first span and behind the last hold NaN, and those that a gap leaves out numbers that no product has."""
    q, k, v, do = _data(2, tq, 2300, 1, 1, 32, 16)
    first = 100 + np.arange(tq) // 700 * 400
    spans = np.stack([first, np.minimum(first + 350, 2250)], 1).astype(np.float32)
    spans[5] = 7, 7
    want = ref.Attention(q, k, v, spans, None, 32 ** -0.5)
    for x in (k, v):
        x[:, :100] = x[:, 2250:] = np.nan
        x[0, 451:499] = 3e4
    out, stat, grads = _run(rt, q, k, v, do, spans=spans)
    ref.assert_within(out, want.out, want.out_tol, "out")
    ref.assert_within(stat, want.stat, want.stat_tol, "statistics")
    for what, got, (value, tol) in zip(("dq", "dk", "dv"), grads, want.backward(out, stat, do)):
        ref.assert_within(got, value, tol, what)
