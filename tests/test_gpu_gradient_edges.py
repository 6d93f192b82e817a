"""Gradients and gated values where few bits or no bits of the answer are left: the sigmoid's slope far from zero, gradient rows
near the largest floats, arguments that are NaN, rows of padding."""
import numpy as np
import pytest
import torch

from sublayer import U8, U24, Weight, close, f64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [336, 333])
def test_sigmoid_slope_keeps_its_bits(dev, n):
    """s(v) s(-v) elementwise relative to itself from -30 to 30, where 1 - s(v) has none of its bits left (rows of zeros: the bias is
    the argument). e^-|v| by the hardware: its argument and the constant of its product with log2 e are a half step each of |v|,
    so 2 |v| half steps, two for the exponential, two for 1 + e, and twice the reciprocal's two, then three products; one rounding to
    bf16."""
    import qmm.ops as ops
    v = torch.linspace(-30, 30, n)
    w, b, one = Weight("q4_0", np.random.default_rng(1), n, 256, dev), v.to(dev), torch.ones(n, device=dev)
    x, s, dy = torch.zeros((3, 256), dtype=torch.float16, device=dev), torch.ones((3, 2), device=dev), torch.ones((3, n), device=dev)
    want = torch.sigmoid(v.double()) * torch.sigmoid(-v.double())
    tol = (1 + U8) * (2 * v.double().abs() + 11) * U24 * want + U8 * want
    _, dpre = ops.linear_backward("q4_0", x, w.w, dy, n, 256, scales=s, bias=b, act="sigmoid")
    _, dgu = ops.ffn_gate_up_backward("q4_0", x, w.w, w.w, dy, n, 256, scales=s, bias=b, bias2=one, act="sigmoid")
    close(f64(dpre), want.expand(3, n), tol.expand(3, n), "dpre")
    close(f64(dgu[:, 0]), want.expand(3, n), tol.expand(3, n), "dg")


@pytest.mark.parametrize("n", [64, 63, 8 * 8193])
def test_gradient_rows_near_the_largest_floats(dev, n):
    """The exponent of a row's scale reaches the largest floats': finite rows stay finite, in [2^13, 2^14) for their largest value."""
    import qmm.ops as ops
    from qmm import _lib
    T, N = 5, -(-n // 64) * 64
    x = torch.from_numpy(np.random.default_rng(2).uniform(-1, 1, (T, 1, n)).astype(np.float32)).to(dev)
    x[:, 0, 0] = 1
    x = x * torch.tensor([2.0 ** 113, 2.0 ** 114, 2.0 ** 117, 2.0 ** 126, 2.0 ** 127], device=dev).reshape(-1, 1, 1)
    x16 = torch.empty((T, 1, N), dtype=torch.float16, device=dev)
    s = torch.empty((T, 2), device=dev)
    _lib.call("qmm_grad_operand", T, 1, n, x.data_ptr(), 0, x16.data_ptr(), s.data_ptr(), ops._stream())
    assert torch.equal(s[:, 1].log2(), torch.tensor([100.0, 101, 104, 113, 114], device=dev)) and (s[:, 0] * s[:, 1] == 1).all()
    assert torch.equal(x16[..., :n], (x * s[:, :1, None]).half()) and (x16[..., n:] == 0).all()
    assert (x16.abs().amax((1, 2)) == 2.0 ** 13).all()
