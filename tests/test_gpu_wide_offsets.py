"""Arrays whose element offsets pass 32 bits: layer norm, the gated product's pointwise part and counter dropout, at both
ends and around 2^31 and 2^32.  The storage is torch's, so that it goes back to the device and not to the library's pool."""
import ctypes

import numpy as np
import pytest

import feed_forward_ref as ref

pytestmark = pytest.mark.gpu


def _over(tensor, shape, first=0):
    """The library's view of ``shape`` from the tensor's element ``first`` on."""
    from tinyflow_amd import ndarray

    class View(ndarray.NDArray):
        __slots__ = ["keep"]
    extents = (ctypes.c_int64 * len(shape))(*shape)
    arr = ndarray.DLArray(tensor.data_ptr() + 4 * first, ndarray.gpu(0), len(shape), extents)
    view = View(ctypes.pointer(arr))
    view.is_freed, view.keep = True, (tensor, extents, arr)
    return view


@pytest.fixture
def room():
    import torch

    def take(count, zeros=False):
        if torch.cuda.mem_get_info()[0] < 4 * count + (1 << 32):
            pytest.skip("the device has no room for %d elements" % count)
        t = (torch.zeros if zeros else torch.empty)(count, device="cuda")
        torch.cuda.synchronize()
        return t
    yield take
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def test_counter_dropout(rt, room):
    import torch
    from tinyflow_amd import gpu_op
    count, some = (1 << 34) + 1026, 4096   # the counter of an element passes 32 bits at 2^34
    t = room(count)
    x = np.random.RandomState(3).normal(0, 1, some).astype(np.float32)
    places = [0, (1 << 31) - 2048, (1 << 32) - 2048, (1 << 34) - 2048]
    for at in places:
        n = min(some, count - at)
        t[at:at + n] = torch.from_numpy(x[:n])
    torch.cuda.synchronize()
    whole = _over(t, (count,))
    gpu_op.counter_dropout(whole, None, whole, 0.5, 77, 1 << 33, rt.stream)
    torch.cuda.synchronize()
    for at in places:
        n = min(some, count - at)
        np.testing.assert_array_equal(t[at:at + n].cpu().numpy(),
                                      np.where(ref.kept(n, 0.5, 77, 1 << 33, at), 2 * x[:n], np.float32(0)))


@pytest.mark.parametrize("cols", [1000, 4100, 20000])
def test_layer_norm(rt, room, cols):
    """Rows of zeros but for five: their y is beta, their dx zero, and nothing of theirs enters the weights' gradients."""
    import torch
    from tinyflow_amd import gpu_op
    rows = (1 << 32) // cols + 2
    picked = [0, 1, (1 << 31) // cols, (1 << 32) // cols, rows - 1]
    rng = np.random.RandomState(cols)
    x, dy = (rng.normal(0, 1, (len(picked), cols)).astype(np.float32) for _ in range(2))
    gamma, beta = ((rng.normal(0, 0.3, cols) + c).astype(np.float32) for c in (1, 0))
    tx, td = room(rows * cols, True), room(rows * cols, True)
    out = room(rows * cols)
    for i, r in enumerate(picked):
        tx[r * cols:(r + 1) * cols] = torch.from_numpy(x[i])
        td[r * cols:(r + 1) * cols] = torch.from_numpy(dy[i])
    small = [torch.from_numpy(v).cuda() for v in (gamma, beta, gamma, beta)]
    torch.cuda.synchronize()
    ax, ad, ao = (_over(t, (rows, cols)) for t in (tx, td, out))
    ag, ab, adg, adb = (_over(t, (cols,)) for t in small)
    gpu_op.layer_norm_forward(ax, ag, ab, ao, 1e-5, rt.stream)
    torch.cuda.synchronize()
    norm = ref.Norm(x, gamma, beta, 1e-5)
    for i, r in enumerate(picked):
        ref.assert_within(out[r * cols:(r + 1) * cols].cpu().numpy(), norm.y[i], norm.y_tol[i], "y of row %d" % r)
    for r in (2, picked[2] + 1, rows - 3):
        np.testing.assert_array_equal(out[r * cols:(r + 1) * cols].cpu().numpy(), beta)
    assert gpu_op.layer_norm_backward(ax, ag, ad, ao, adg, adb, 1e-5, rt.stream) == 0
    torch.cuda.synchronize()
    (dx, dx_tol), *weights = norm.backward(dy)
    for i, r in enumerate(picked):
        ref.assert_within(out[r * cols:(r + 1) * cols].cpu().numpy(), dx[i], dx_tol[i], "dx of row %d" % r)
    for r in (2, picked[2] + 1, rows - 3):
        assert not out[r * cols:(r + 1) * cols].cpu().numpy().any()
    for got, (value, tol), what in zip(small[2:], weights, ("dgamma", "dbeta")):
        ref.assert_within(got.cpu().numpy(), value, tol, what)


def test_pointwise_calls(rt, room):
    import torch
    from tinyflow_amd import gpu_op
    count, some = (1 << 32) + 1027, 1024
    pre, h = room(2 * count), room(count)
    rng = np.random.RandomState(8)
    g, u, d = (rng.normal(0, 1, some).astype(np.float32) for _ in range(3))
    places = [0, (1 << 31) - 512, count - some]
    for at in places:
        pre[at:at + some] = torch.from_numpy(g)
        pre[count + at:count + at + some] = torch.from_numpy(u)
    torch.cuda.synchronize()
    ap, ah = _over(pre, (2, count)), _over(h, (count,))
    gpu_op.gated_activation(ap, ah, "silu", rt.stream)
    torch.cuda.synchronize()
    (act, _, _), ends = ref.act_and_slope(g.astype(np.float64), "silu"), [h[at:at + some].cpu().numpy() for at in places]
    for got in ends:
        ref.assert_within(got, act * u, 12 * ref.U * np.abs(g * u), "h")
    for at in places:
        h[at:at + some] = torch.from_numpy(d)
    torch.cuda.synchronize()
    gpu_op.gated_activation_backward(ap, ah, ap, "silu", rt.stream)   # in place
    torch.cuda.synchronize()
    value, tol = ref.pointwise_gradient(np.stack([g, u]), d, "silu")
    for at in places:
        got = [pre[first + at:first + at + some].cpu().numpy() for first in (0, count)]
        ref.assert_within(np.stack(got), value, tol, "gradients")


@pytest.mark.parametrize("m,k,f", [(131075, 40, 4090), (131075, 4090, 40), (3, 23010, 23010), (20, 23010, 23010), (2, 2500, 214000),
                                   (140, 23010, 23010), (1 << 22, 2, 7), (1 << 26, 1, 7), (1, 7, 1 << 26)])
def test_gated_feed_forward_next_to_2_gib(rt, room, m, k, f):
    """Zeros but for rows, columns and elements of the reduction at both ends and in the middle."""
    import torch
    from tinyflow_amd import gpu_op
    rows, along, cols = ([0, n // 2, n - 1] if n > 2 else list(range(n)) for n in (m, k, f))
    rng = np.random.RandomState(m % 1000 + k + f % 1000)
    x, gate, up, dh = (rng.normal(0, 1, s).astype(np.float32) for s in ((len(rows), len(along)), (len(along), len(cols)),
                                                                     (len(along), len(cols)), (len(rows), len(cols))))
    shapes = {"x": (m, k), "gate": (k, f), "up": (k, f), "pre": (2, m, f), "h": (m, f), "dx": (m, k), "dgate": (k, f), "dup": (k, f)}
    t = {name: room(int(np.prod(shape)), zeros=True).view(shape) for name, shape in shapes.items()}
    at = {"x": (rows, along), "gate": (along, cols), "up": (along, cols), "h": (rows, cols), "dx": (rows, along),
          "dgate": (along, cols), "dup": (along, cols)}

    def picked(name):
        r, c = (torch.tensor(i, device="cuda") for i in at[name])
        return r[:, None], c[None, :]

    def read(name):
        return t[name][picked(name)].cpu().numpy()

    for name, value in (("x", x), ("gate", gate), ("up", up)):
        t[name][picked(name)] = torch.from_numpy(value).cuda()
    torch.cuda.synchronize()
    a = {name: _over(v, shapes[name]) for name, v in t.items()}
    assert gpu_op.gated_feed_forward(a["x"], a["gate"], a["up"], a["pre"], a["h"], "silu", rt.stream) == 0
    torch.cuda.synchronize()
    (pre, d_pre), (h, d_h) = ref.gated(x, gate, up, "silu")
    ref.assert_within(read("h"), h, d_h, "h")
    r, c = picked("h")
    got = np.stack([t["pre"][half][r, c].cpu().numpy() for half in range(2)])
    ref.assert_within(got, pre, d_pre, "pre")
    assert int(torch.count_nonzero(t["h"])) == np.count_nonzero(read("h"))   # nothing elsewhere
    t["h"].zero_()
    t["h"][picked("h")] = torch.from_numpy(dh).cuda()
    torch.cuda.synchronize()
    if m == 1 << 26:
        return   # scratch of 40 GB, which the pool would keep
    assert gpu_op.gated_feed_forward_backward(a["x"], a["gate"], a["up"], a["pre"], a["h"], a["dx"], a["dgate"], a["dup"], "silu",
                                              rt.stream) == 0
    torch.cuda.synchronize()
    (dpre, d_dpre) = ref.pointwise_gradient(got.astype(np.float64), dh, "silu")
    for name, (value, tol) in zip(("dx", "dgate", "dup"), ref.gated_backward(x, gate, up, dpre, d_dpre)):
        ref.assert_within(read(name), value, tol, name)
        assert int(torch.count_nonzero(t[name])) == np.count_nonzero(read(name)), name
