"""The largest number of rows that the norms and the gradient operand take: more workgroups than one dimension of a grid holds."""
import pytest
import torch

from sublayer import U24

pytestmark = pytest.mark.gpu
ROWS = 1 << 24
EPS = 1e-6


def _parts(rows):
    return [slice(0, 700), slice(rows // 2 - 350, rows // 2 + 350), slice(rows - 700, rows)]


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("k,out", [(8, "bf16"), (9, "bf16"), (9, "f16"), (32, "q8"), (520, "bf16")])
def test_rms_norm(dev, k, out):
    import qmm.ops as ops
    x = torch.empty((ROWS, k), dtype=torch.bfloat16, device=dev).normal_()
    w = 1 + 0.1 * torch.randn(k, device=dev)
    y, scales, _ = ops.rms_norm(x, w, EPS, out=out)
    for p in _parts(ROWS):
        want, ws, _ = ops.rms_norm(x[p].clone(), w, EPS, out=out)
        if out == "q8":
            assert torch.equal(y[p.start * k:p.stop * k], want[:700 * k])
            got = y[ROWS * k:].view(torch.float32).view(ROWS, -1)[p]
            assert torch.equal(got, want[700 * k:].view(torch.float32).view(700, -1))
        else:
            assert torch.equal(y[p], want) and (scales is None or torch.equal(scales[p], ws))


@pytest.mark.parametrize("k", [8, 9, 136])
def test_rms_norm_backward(dev, k):
    """dweight: rows up to ROWS / 128 on a thread's chain and 100 additions that join them, each a half step of the sum of |terms|."""
    import qmm.ops as ops
    h = torch.empty((ROWS, k), dtype=torch.bfloat16, device=dev).normal_()
    dy = torch.empty((ROWS, k), dtype=torch.bfloat16, device=dev).normal_()
    w = 1 + 0.1 * torch.randn(k, device=dev)
    dx, dw = ops.rms_norm_backward(h, w, dy, EPS)
    for p in _parts(ROWS):
        assert torch.equal(dx[p], ops.rms_norm_backward(h[p].clone(), w, dy[p].clone(), EPS, dweight=False)[0])
    assert torch.equal(ops.rms_norm_backward(h, w, dy, EPS, dweight=False)[0], dx)
    want, mag = torch.zeros(k, dtype=torch.float64, device=dev), torch.zeros(k, dtype=torch.float64, device=dev)
    for a in range(0, ROWS, ROWS // 16):
        hd = h[a:a + ROWS // 16].double()
        t = dy[a:a + ROWS // 16].double() * hd / torch.sqrt(hd.square().mean(-1, keepdim=True) + EPS)
        want += t.sum(0)
        mag += t.abs().sum(0)
    assert ((dw.double() - want).abs() <= (ROWS / 128 + 100) * U24 * mag).all()


@pytest.mark.parametrize("n", [8, 9])
def test_grad_operand(dev, n):
    import qmm.ops as ops
    from qmm import _lib

    def operand(x):
        T = x.shape[0]
        x16, s = torch.empty((T, 64), dtype=torch.float16, device=dev), torch.empty((T, 2), device=dev)
        _lib.call("qmm_grad_operand", T, 1, n, x.data_ptr(), 2, x16.data_ptr(), s.data_ptr(), ops._stream())
        return x16, s

    x = torch.empty((ROWS, n), dtype=torch.bfloat16, device=dev).normal_()
    x16, s = operand(x)
    for p in _parts(ROWS):
        want, ws = operand(x[p].clone())
        assert torch.equal(x16[p], want) and torch.equal(s[p], ws)
