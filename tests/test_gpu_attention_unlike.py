"""Attention of operands whose rows or columns differ by powers of ten: what is small has its own digits.  The small part is compared with a reference
that does not know of the large one, so that no bound is of the large one's size."""
import numpy as np
import pytest

import attention_ref as ref
from test_gpu_attention import _check, _data, _run

pytestmark = pytest.mark.gpu


def _off(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


# a row of a result is a sum of up to 300 products of sums of 64: each rounding 2^-24 of a magnitude that cancellation makes up to four times the
# result's: 2^-24 (300 + 64) 4 < 2^-13.4
ROW = 2.0 ** -13.4


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("power", [8, 16, 24, 30, 40, 60])
def test_a_query_among_larger_ones(rt, monkeypatch, split, power):
    """Every 32nd query is 2^power of the others."""
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    q, k, v, do = _data(1, 320, 512, 2, 1, 64, 31)
    large = np.arange(320) % 32 == 9
    q[:, large] *= np.float32(2.0 ** power)
    out, stat, (dq, _, _) = _run(rt, q, k, v, do)
    want = ref.Attention(q[:, ~large], k, v, None, None, 0.125)
    ref.assert_within(out[:, ~large], want.out, want.out_tol, "out")
    ref.assert_within(stat[..., ~large], want.stat, want.stat_tol, "statistics")
    value, tol = want.backward(out[:, ~large], stat[..., ~large], do[:, ~large])[0]
    ref.assert_within(dq[:, ~large], value, tol, "dq")


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("power", [-12, -30, -60])
def test_queries_of_documents(rt, monkeypatch, split, power):
    """Documents that end inside of blocks, every other one with queries of 2^power: their keys' gradients are as small."""
    from tinyflow_amd import gpu_op
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    q, k, v, do = _data(1, 320, 320, 2, 2, 64, 32)
    documents = np.arange(320) // 80
    q[:, documents % 2 == 1] *= np.float32(2.0 ** power)
    spans = gpu_op.attention_spans(320, documents=documents)
    out, stat, (_, dk, _) = _run(rt, q, k, v, do, spans=spans)
    for n in range(4):
        own = documents == n
        want = ref.Attention(q[:, own], k[:, own], v[:, own], None, None, 0.125).backward(out[:, own], stat[:, :, own], do[:, own])[1][0]
        assert _off(dk[:, own], want) <= ROW, "dk of document %d" % n


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("power", [14, 24, 30, 40])
@pytest.mark.parametrize("which", ["query", "key"])
def test_a_large_column_that_meets_zeros(rt, monkeypatch, split, power, which):
    """The scores come from the other columns."""
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    q, k, v, do = _data(1, 300, 300, 2, 1, 64, 33)
    one, other = (q, k) if which == "query" else (k, q)
    one[..., 0] *= np.float32(2.0 ** power)
    other[..., 0] = 0
    out, stat, grads = _run(rt, q, k, v, do, causal=True)
    want = ref.Attention(q[..., 1:], k[..., 1:], v, None, None, 0.125, causal=True)
    ref.assert_within(out, want.out, want.out_tol, "out")
    ref.assert_within(stat, want.stat, want.stat_tol, "statistics")
    values = want.backward(out, stat, do)
    for what, got, (value, tol) in zip(("dq", "dk"), grads, values):
        ref.assert_within(got[..., 1:], value, tol, what)
    ref.assert_within(grads[2], *values[2], "dv")


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("power", [14, 24, 30, 40])
def test_a_large_column_of_values(rt, monkeypatch, split, power):
    """The other columns' outputs, and with no gradient in the large column all other gradients."""
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    q, k, v, do = _data(1, 300, 300, 2, 1, 64, 34)
    v[..., 5] *= np.float32(2.0 ** power)
    do[..., 5] = 0
    out, stat, grads = _run(rt, q, k, v, do, causal=True)
    rest = np.arange(64) != 5
    want = ref.Attention(q, k, v[..., rest], None, None, 0.125, causal=True)
    ref.assert_within(out[..., rest], want.out, want.out_tol, "out")
    # scores are of 64 columns, dp of the 63 that count
    assert _off(out[..., 5], ref.Attention(q, k, v[..., 5:6], None, None, 0.125, causal=True).out[..., 0]) <= ROW
    small = want.backward(out[..., rest], stat, do[..., rest])
    for what, got, (value, tol) in zip(("dq", "dk"), grads, small):
        ref.assert_within(got, value, tol, what)
    ref.assert_within(grads[2][..., rest], *small[2], "dv")


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("power", [-24, -34, -44])
@pytest.mark.parametrize("which", range(4))
def test_a_small_column(rt, monkeypatch, split, power, which):
    """Its own gradient (of a query's or key's column, from the other's; of a value's, from the output's) or output has its digits."""
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    a = _data(1, 300, 300, 2, 1, 64, 35)
    a[which][..., 7] *= np.float32(2.0 ** power)
    q, k, v, do = a
    out, stat, grads = _run(rt, q, k, v, do, causal=True)
    want = ref.Attention(q, k, v, None, None, 0.125, causal=True)
    values = [value for value, _ in want.backward(out, stat, do)]
    pairs = {0: (grads[1], values[1]), 1: (grads[0], values[0]), 2: (out, want.out), 3: (grads[2], values[2])}
    got, value = pairs[which]
    assert _off(got[..., 7], value[..., 7]) <= ROW


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("d", [48, 64, 128])
@pytest.mark.parametrize("power", [20, 32, 40, 60])
def test_keys_that_every_query_gives_little(rt, monkeypatch, split, d, power):
    """A share of about 2^-power each: their values' and their own gradients are as small, and have their digits."""
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    q, k, v, do = _data(1, 300, 300, 2, 1, d, 36)
    low = np.arange(300) // 7 % 3 == 1
    q[..., 0] = 4
    k[..., 0] = 0
    k[:, low, :, 0] = -power * np.log(2) * np.sqrt(d) / 4
    out, stat, (_, dk, dv) = _run(rt, q, k, v, do)
    want = ref.Attention(q, k, v, None, None, d ** -0.5).backward(out, stat, do)
    # Scores of up to 42 and 10 are sums of up to 128 products in chains of 40: 2^-24 40 52 off, and as much of the share: 2^-13; the sums themselves as
    # above.
    for what, got, value in (("dk", dk, want[1][0]), ("dv", dv, want[2][0])):
        assert _off(got[:, low], value[:, low]) <= 2.0 ** -12.4, what


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("power", [-90, -105, -116])
def test_small_values_everywhere(rt, monkeypatch, split, power):
    """All values, or all gradients, near the smallest that fp32 has."""
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    q, k, v, do = _data(1, 300, 300, 2, 1, 64, 37)
    small = np.float32(2.0 ** power)
    tiny = 300 * 2.0 ** -149   # what is lost below the normal numbers
    want = ref.Attention(q, k, v * small, None, None, 0.125, causal=True)
    out, stat, grads = _run(rt, q, k, v * small, do * np.float32(64), causal=True)
    ref.assert_within(out, want.out, want.out_tol + tiny, "out")
    want = ref.Attention(q, k, v, None, None, 0.125, causal=True)
    out, stat, grads = _run(rt, q, k, v, do * small, causal=True)
    for what, got, (value, tol) in zip(("dq", "dk", "dv"), grads, want.backward(out, stat, do * small)):
        ref.assert_within(got, value, tol + 64 * tiny, what)


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("scale", [1e3, 1e6, 1e9])
def test_scores_that_pass_every_digit(rt, monkeypatch, split, scale):
    """Every query has one key that takes all: scores of up to 1e10, whose differences are what they are."""
    from tinyflow_amd import gpu_op, ndarray
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    rng = np.random.RandomState(38)
    n, d = 256, 64
    # whole numbers: scores are exact in fp32, and the statistic is the largest one's
    q = rng.randint(-3, 4, (1, n, 1, d)).astype(np.float32)
    k = rng.randint(-3, 4, (1, n, 1, d)).astype(np.float32)
    v, do = (rng.normal(0, 1, (1, n, 1, d)).astype(np.float32) for _ in range(2))
    scale = float(2.0 ** np.round(np.log2(scale)))
    a = [ndarray.array(x, ctx=rt.ctx) for x in (q, k, v, do)]
    out, stat, dq, dk, dv = (ndarray.array(np.full(s, 7.25, np.float32), ctx=rt.ctx) for s in (q.shape, (1, 1, n)) + (q.shape,) * 3)
    numbers = (1, 1, 1, scale, 0.0, False, rt.stream)
    assert gpu_op.attention_forward(*a[:3], None, None, out, stat, *numbers) == 0
    assert gpu_op.attention_backward(*a[:3], None, None, out, stat, a[3], dq, dk, dv, *numbers) == 0
    s = (q[0, :, 0] @ k[0, :, 0].T).astype(np.float64)
    p = (s == s.max(1, keepdims=True)) / (s == s.max(1, keepdims=True)).sum(1, keepdims=True)
    assert np.abs(out.asnumpy()[0, :, 0] - p @ v[0, :, 0]).max() <= 2.0 ** -18   # sums of a few values of up to 4
    for got in (dq, dk, dv):
        assert np.isfinite(got.asnumpy()).all()


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("small,scale", [((-60, -20), 38), ((-50, -35), 39), ((-20, -15), 35), ((20, 10), -30)])
def test_scales_that_make_up_for_small_operands(rt, monkeypatch, split, small, scale):
    """Queries and keys of 2^small with a scale of 2^scale."""
    from tinyflow_amd import gpu_op, ndarray
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    q, k, v, do = _data(1, 300, 300, 2, 1, 64, 39)
    q, k = q * np.float32(2.0 ** small[0]), k * np.float32(2.0 ** small[1])
    scale = 2.0 ** scale
    a = [ndarray.array(x, ctx=rt.ctx) for x in (q, k, v, do)]
    out, stat, *grads = (ndarray.array(np.full(s, 7.25, np.float32), ctx=rt.ctx) for s in (q.shape, (1, 2, 300), q.shape, k.shape, v.shape))
    numbers = (1, 2, 1, scale, 0.0, False, rt.stream)
    assert gpu_op.attention_forward(*a[:3], None, None, out, stat, *numbers) == 0
    assert gpu_op.attention_backward(*a[:3], None, None, out, stat, a[3], *grads, *numbers) == 0
    want = ref.Attention(q, k, v, None, None, scale)
    ref.assert_within(out.asnumpy(), want.out, want.out_tol, "out")
    ref.assert_within(stat.asnumpy(), want.stat, want.stat_tol, "statistics")
    for what, got, (value, tol) in zip(("dq", "dk", "dv"), grads, want.backward(out.asnumpy(), stat.asnumpy(), do)):
        ref.assert_within(got.asnumpy(), value, tol, what)


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("power", [12, 30, 50])
@pytest.mark.parametrize("which", ["values", "gradients"])
def test_neighbours_with_larger_numbers(rt, monkeypatch, split, power, which):
    """Two documents whose border is no border of a block of queries (of keys), the first with values (gradients) of 2^power of the second's: the
    second's results are those that it has alone."""
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    tq, tk, rows, keys = (300, 320, 40, 64) if which == "values" else (320, 300, 64, 40)
    q, k, v, do = _data(1, tq, tk, 2, 2, 64, 40)
    spans = np.zeros((tq, 2), np.float32)
    spans[:rows, 1] = keys
    spans[rows:] = keys, tk
    if which == "values":
        v[:, :keys] *= np.float32(2.0 ** power)
    else:
        do[:, :rows] *= np.float32(2.0 ** power)
    out, stat, (dq, dk, dv) = _run(rt, q, k, v, do, spans=spans)
    want = ref.Attention(q[:, rows:], k[:, keys:], v[:, keys:], None, None, 0.125)
    ref.assert_within(out[:, rows:], want.out, want.out_tol, "out")
    ref.assert_within(stat[..., rows:], want.stat, want.stat_tol, "statistics")
    values = want.backward(out[:, rows:], stat[..., rows:], do[:, rows:])
    for what, got, (value, tol) in zip(("dq", "dk", "dv"), (dq[:, rows:], dk[:, keys:], dv[:, keys:]), values):
        ref.assert_within(got, value, tol, what)


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("power", [12, 30, 50])
@pytest.mark.parametrize("first", [True, False])
def test_large_values_of_which_little_is_taken(rt, monkeypatch, split, power, first):
    """A block of keys with values of 2^power, and a share of 2^-power 2^-12 for each of its keys: outputs and gradients come from the others."""
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    q, k, v, do = _data(1, 200, 320, 2, 1, 64, 41)
    block = slice(0, 32) if first else slice(224, 256)
    q[..., 0], k[..., 0] = 4, 0
    k[:, block, :, 0] = -(power + 12) * np.log(2) * 8 / 4
    v[:, block] *= np.float32(2.0 ** power)
    out, stat, grads = _run(rt, q, k, v, do)
    want = ref.Attention(q, k, v, None, None, 0.125)
    for what, got, value in zip(("out", "dq", "dk", "dv"), [out] + grads, [want.out] + [x for x, _ in want.backward(out, stat, do)]):
        # the shares of the block are of scores of up to 44: 2^-24 40 52 off, and so are their dk and dv
        assert _off(got, value) <= 2.0 ** -12.4, what
        if what in ("dk", "dv"):
            assert _off(got[:, block], value[:, block]) <= 2.0 ** -12.4, what


def test_a_scale_that_only_a_cap_bears(rt):
    """Scores past every digit under a cap: each is the cap, or its opposite."""
    from tinyflow_amd import gpu_op, ndarray
    rng = np.random.RandomState(42)
    q, k = (np.sign(rng.normal(0, 1, (1, 256, 1, 64))).astype(np.float32) for _ in range(2))
    q[..., 0] *= 1.5   # no product is 0
    v = rng.normal(0, 1, (1, 256, 1, 64)).astype(np.float32)
    a = [ndarray.array(x, ctx=rt.ctx) for x in (q, k, v)]
    out = ndarray.array(np.full(q.shape, 7.25, np.float32), ctx=rt.ctx)
    assert gpu_op.attention_forward(*a, None, None, out, None, 1, 1, 1, 1e37, 1e30, False, rt.stream) == 0
    # exp2 of a difference of 2e30 is 0, of none 1
    above = (q[0, :, 0].astype(np.float64) @ k[0, :, 0].T.astype(np.float64)) > 0
    want = above @ v[0, :, 0].astype(np.float64) / above.sum(1, keepdims=True)
    assert np.abs(out.asnumpy()[0, :, 0] - want).max() <= 300 * 2.0 ** -24 * 4   # sums of up to 256 values of up to 4


@pytest.mark.parametrize("distance", [False, True])
def test_errors_are_those_of_fp32(rt, monkeypatch, distance):
    """Gradients of documents, whose shares grow by powers of ten on the way through the rows.  A pair's elements are off by 2^-24.8 in the mean, two of them and
    the product left out by 2^-23.5, an fp32 product and its sum by as much; the rest both engines have: the errors' ratio is at most that of one
    such error and of two, the square root of two, and is given a tenth for chance."""
    from tinyflow_amd import gpu_op
    q, k, v, do = _data(2, 1001, 1001, 4, 2, 72, 43)
    documents = np.repeat(np.arange(4), [100, 201, 300, 400])[None].repeat(2, 0)
    spans = gpu_op.attention_spans(1001, documents=documents, causal=True)
    slopes = 2.0 ** (-2.0 * np.arange(1, 5)) if distance else None
    want = ref.Attention(q, k, v, spans, slopes, 72 ** -0.5)
    off = {}
    for split in ("0", "1"):
        monkeypatch.setenv("TINYFLOW_SPLIT", split)
        out, stat, grads = _run(rt, q, k, v, do, spans=spans, slopes=slopes)
        values = [want.out] + [value for value, _ in want.backward(want.out, want.stat, do)]
        off[split] = [_off(got, value) for got, value in zip([out] + grads, values)]
    for what, ours, fp32 in zip(("out", "dq", "dk", "dv"), off["1"], off["0"]):
        assert ours <= 1.55 * fp32, "%s is %.2g off, %.2g on the fp32 instruction" % (what, ours, fp32)


@pytest.mark.parametrize("split", ["0", "1"])
@pytest.mark.parametrize("power", [80, 95, 105])
def test_shares_near_the_smallest_numbers(rt, monkeypatch, split, power):
    """Keys that every query gives 2^-power: dv is as small, and has its digits."""
    monkeypatch.setenv("TINYFLOW_SPLIT", split)
    q, k, v, do = _data(1, 200, 300, 2, 1, 64, 44)
    low = np.arange(300) % 11 == 3
    q[..., 0], k[..., 0] = 4, 0
    k[:, low, :, 0] = -power * np.log(2) * 8 / 4
    do *= np.float32(100)
    out, stat, (_, _, dv) = _run(rt, q, k, v, do)
    value = ref.Attention(q, k, v, None, None, 0.125).backward(out, stat, do)[2][0]
    # scores of up to 73 and 10: 2^-24 40 83 off, and so are shares: 2^-12.3
    assert _off(dv[:, low], value[:, low]) <= 2.0 ** -12
