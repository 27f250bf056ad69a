"""What the gated product asks for beside its arrays, and calls under capture."""
import ctypes

import numpy as np
import pytest

import feed_forward_ref as ref
from test_gpu_gated import _data
from test_gpu_wide_offsets import _over, room  # noqa: F401

pytestmark = pytest.mark.gpu


def _arrays(rt, *values):
    from tinyflow_amd import ndarray
    return [ndarray.array(np.ascontiguousarray(v, np.float32), ctx=rt.ctx) for v in values]


# many rows of a few columns, which blocks of 32 of the reduction would hold several times over
@pytest.mark.parametrize("m,k,f", [(1 << 19, 1, 7), (1 << 18, 7, 1), ((1 << 18) + 5, 3, 5), (100003, 8, 9)])
def test_narrow_extents_take_no_more_than_their_arrays(rt, m, k, f):
    from tinyflow_amd import gpu_op
    x, gate, up, dh = _data(m, k, f, 3)
    pre = np.stack([x @ gate, x @ up])
    arrays = _arrays(rt, x, gate, up, pre, dh)
    out = _arrays(rt, *(np.full(v.shape, 7.25) for v in (x, gate, up)))
    used = gpu_op.device_memory_stats()[1]
    try:
        gpu_op.set_device_memory_limit(used + 4 * (x.size + 3 * dh.size))
        assert gpu_op.gated_feed_forward_backward(*arrays, *out, "silu", rt.stream) == 0
        got = [a.asnumpy() for a in out]
    finally:
        gpu_op.set_device_memory_limit(0)
    dpre, d_dpre = ref.pointwise_gradient(pre, dh, "silu")
    for what, a, (value, tol) in zip(("dx", "dgate", "dup"), got, ref.gated_backward(x, gate, up, dpre, d_dpre)):
        ref.assert_within(a, value, tol, what)


def test_the_most_rows_there_are(rt, room):  # noqa: F811
    """The backward pass of 2^26 rows: zeros but for rows at both ends and in the middle."""
    import torch
    from tinyflow_amd import gpu_op
    m, k, f = 1 << 26, 1, 7
    rows = [0, 1, m // 2, m - 33, m - 1]
    rng = np.random.RandomState(9)
    x, dh = rng.normal(0, 1, (len(rows), k)).astype(np.float32), rng.normal(0, 1, (len(rows), f)).astype(np.float32)
    gate, up = (rng.normal(0, 1, (k, f)).astype(np.float32) for _ in range(2))
    pre = np.stack([x @ gate, x @ up])
    tx, tdx = room(m * k, True).view(m, k), room(m * k).view(m, k)
    tpre, tdh = room(2 * m * f, True).view(2, m, f), room(m * f, True).view(m, f)
    at = torch.tensor(rows, device="cuda")
    tx[at], tdh[at] = torch.from_numpy(x).cuda(), torch.from_numpy(dh).cuda()
    tpre[:, at] = torch.from_numpy(pre).cuda()
    tdx.fill_(7.25)
    torch.cuda.synchronize()
    ag, au, dgate, dup = _arrays(rt, gate, up, gate, up)
    before = gpu_op.device_memory_stats(reset_peak=True)[1]
    assert gpu_op.gated_feed_forward_backward(_over(tx, (m, k)), ag, au, _over(tpre, (2, m, f)), _over(tdh, (m, f)),
                                              _over(tdx, (m, k)), dgate, dup, "silu", rt.stream) == 0
    torch.cuda.synchronize()
    assert gpu_op.device_memory_stats()[2] - before <= 4 * m * (k + 3 * f)
    dpre, d_dpre = ref.pointwise_gradient(pre, dh, "silu")
    (dx, dx_tol), *weights = ref.gated_backward(x, gate, up, dpre, d_dpre)
    ref.assert_within(tdx[at].cpu().numpy(), dx, dx_tol, "dx")
    assert int(torch.count_nonzero(tdx)) == np.count_nonzero(tdx[at].cpu().numpy())
    for got, (value, tol), what in zip((dgate, dup), weights, ("dgate", "dup")):
        ref.assert_within(got.asnumpy(), value, tol, what)


def test_a_captured_graph(rt):
    """Calls in registers that take no scratch replay; those that fold or run on pairs are refused, and leave the capture as it is."""
    import torch
    from tinyflow_amd import gpu_op
    stream = gpu_op.create_cudaStream()
    kept, refused = [], []
    for m, k, f in [(9, 40, 65), (70, 40, 8300), (927, 34, 2382), (4, 2560, 96), (2, 2000, 300)]:   # one piece; a strip a wave; few rows
        x, gate, up, _ = _data(m, k, f, m)
        kept.append((_arrays(rt, x, gate, up, np.full((2, m, f), 7.25), np.full((m, f), 7.25)), (m, k, f)))
    for m, k, f in [(24, 300, 520), (4, 2600, 64), (1100, 1030, 700)]:   # in pieces; on pairs
        x, gate, up, _ = _data(m, k, f, m)
        refused.append(_arrays(rt, x, gate, up, np.full((2, m, f), 7.25), np.full((m, f), 7.25)))

    def calls():
        for a, _ in kept:
            assert gpu_op.gated_feed_forward(*a, "silu", stream) == 0
    calls()
    for a in refused:
        assert gpu_op.gated_feed_forward(*a, "silu", stream) == 0
        gpu_op.array_set(a[4], 7.25, stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    external = torch.cuda.ExternalStream(ctypes.cast(stream.contents, ctypes.c_void_p).value)
    with torch.cuda.graph(graph, stream=external):
        calls()
        for a in refused:
            with pytest.raises(RuntimeError):
                gpu_op.gated_feed_forward(*a, "silu", stream)
    for replay in range(3):
        values = []
        for a, (m, k, f) in kept:
            x, gate, up, _ = _data(m, k, f, 100 + replay)
            a[0][:], a[1][:], a[2][:] = x, gate, up
            values.append((x, gate, up))
            gpu_op.array_set(a[3], 7.25, stream)
            gpu_op.array_set(a[4], 7.25, stream)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [(a[3].asnumpy(), a[4].asnumpy()) for a, _ in kept]
        for (pre, h), v in zip(got, values):
            (pre_ref, pre_tol), (h_ref, h_tol) = ref.gated(*v, "silu")
            ref.assert_within(pre, pre_ref, pre_tol, "pre")
            ref.assert_within(h, h_ref, h_tol, "h")
        calls()
        for (pre, h), (a, _) in zip(got, kept):
            np.testing.assert_array_equal(pre, a[3].asnumpy())
            np.testing.assert_array_equal(h, a[4].asnumpy())
    for a in refused:
        assert (a[4].asnumpy() == np.float32(7.25)).all()
    gpu_op.destroy_cudaStream(stream)
