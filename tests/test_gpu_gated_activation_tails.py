"""Activations of large negative arguments, relative to themselves, within what the header states.

Sigmoid: the exponent -x log2(e) is off by 2^-24 of it and by what the constant's rounding is, 2^-26, which carried through
exp2 is |x| (2^-24 + 2^-26) of the result; exp2 and the reciprocal are right to one step of 2^-23, the sum and SiLU's product are
rounded once: 3 * 2^-23.  GELU: the fitted tail is off by 2.6e-5 of itself from -4 down, 1.8e-7 of 1 anywhere."""
import numpy as np
import pytest
from scipy.special import expit, ndtr

pytestmark = pytest.mark.gpu


def _activation(rt, x, activation):
    from tinyflow_amd import gpu_op, ndarray
    pre = ndarray.array(np.stack([x, np.ones_like(x)]), ctx=rt.ctx)
    h = ndarray.array(np.full_like(x, 7.25), ctx=rt.ctx)
    gpu_op.gated_activation(pre, h, activation, rt.stream)
    return h.asnumpy().astype(np.float64)


@pytest.mark.parametrize("activation", ["sigmoid", "silu"])
def test_exponential_tails(rt, activation):
    x = np.linspace(-86, 0, 300007).astype(np.float32)[:-1]
    wide = x.astype(np.float64)
    value = expit(wide) * (wide if activation == "silu" else 1)
    off = np.abs(_activation(rt, x, activation) - value) / np.abs(value)
    assert (off <= 2.0 ** -21 + np.abs(wide) * 2.0 ** -23).all()
    far = np.float32([-90, -200, -1e30, -3e38])
    assert (np.abs(_activation(rt, far, activation)) < 1e-35).all()


def test_the_normal_distributions_tail(rt):
    x = np.concatenate([np.linspace(-12.9, 0, 300007)[:-1], np.linspace(0, 30, 50001), [1e20, 3e38]]).astype(np.float32)
    wide = x.astype(np.float64)
    value = wide * ndtr(wide)
    off = np.abs(_activation(rt, x, "gelu") - value)
    assert (off <= np.abs(wide) * 2.0 ** -21).all()
    assert (off <= 4e-5 * np.abs(value))[x < 0].all()
    far = np.float32([-14, -100, -1e30, -3e38])
    assert (np.abs(_activation(rt, far, "gelu")) < 1e-35).all()
