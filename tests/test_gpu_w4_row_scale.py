"""Many rows of 4-bit products: rows of any size keep f16's eleven bits on their way into the GEMM and its transposed form."""
import pytest
import torch

from qmm import _lib, ops
from ragged_case import U, gen, held, w4_raw
from test_gpu_w4 import ROW, packed, row_rounding

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("rows,n,k,group", [(100, 40, 640, 64), (70, 33, 8192, ROW), (300, 264, 160, 32)])
@pytest.mark.parametrize("x_type", ["bf16", "f32"])
@pytest.mark.parametrize("size", [2.0 ** 127, 2.0 ** 100, 2.0 ** -12, 2.0 ** -21, 2.0 ** -60, 2.0 ** -100])
def test_many_rows_of_any_size(dev, rows, n, k, group, x_type, size):
    """The products through the row scale and the gradient operand, whose rows enter as f16 times a power of two."""
    g = gen(rows + n)
    q, s, z, _, _ = w4_raw(g, n, k, group)
    s = (s.float() / 64).half()
    at = torch.arange(k) // group
    w = s.double()[:, at] * (q.double() - z.double()[:, at])
    wp, ws = packed((q, s, z), group, dev)
    x, dy = (((torch.rand((rows, c), generator=g) * 1.75 - 0.875).double() * size).to(T[x_type]) for c in (k, n))
    tiny = 2.0 ** -149   # a subnormal result's step
    # weights below f16's smallest normal value are its multiples of 2^-24 as s is, so that their products' rounding is 2^-11 of them at most
    for y, a, b, terms, width in ((ops.w4_mm(x.to(dev), wp, ws, n, k, group, out_dtype=torch.float32), x.double(), w.t(), x.double().abs() @ w.abs().t(), k),
                                  (ops.w4_mm_t(dy.to(dev), wp, ws, n, k, group, out_dtype=torch.float32), dy.double(), w, dy.double().abs() @ w.abs(), n)):
        assert y.isfinite().all()
        held(y, a @ b, (2.0 ** -11 + width * U) * terms + row_rounding(a.to(T[x_type]), b.abs().sum(0), terms) + tiny)


@pytest.mark.parametrize("k", [8, 40, 333, 1000, 4096, 8200, 12288, 16384, 20000, 40000])   # each kernel of the row scale
@pytest.mark.parametrize("x_type", ["bf16", "f32"])
def test_operand(dev, k, x_type):
    """A power of two a row that brings its largest value to 2^13 .. 2^14, every value rounded once; zero, subnormal and infinite rows."""
    size = torch.tensor([127, 116, 100, 13, 0, -14, -30, -75, -112, -113, -120, -126, 0, 0, 0, 0])
    g, rows = gen(k), len(size)
    x = ((torch.rand((rows, k), generator=g) * 1.75 - 0.875) * torch.exp2(size.float())[:, None]).to(T[x_type])
    x[12] = 0
    x[13, ::2] = float("nan")
    x[14, k - 1] = float("inf")
    x[15] = 2.0 ** -130
    xd = x.to(dev)
    x16, s = torch.full((rows + 1, k), 9.0, dtype=torch.float16, device=dev), torch.empty((rows, 2), device=dev)
    _lib.call("qmm_row_scale_f16_wide", rows, k, xd.data_ptr(), ops._dt(xd), s.data_ptr(), x16.data_ptr(), ops._stream())
    assert (x16[rows] == 9).all()
    x16, s = x16[:rows].cpu(), s.cpu().double()
    assert torch.equal(s[:, 0] * s[:, 1], torch.ones(rows, dtype=torch.float64)) and (torch.frexp(s[:, 0]).mantissa == 0.5).all()
    exact = x.double() * s[:, :1]
    keep = [r for r in range(rows) if r not in (13, 14)]
    assert torch.equal(x16[keep], exact[keep].half())
    m = exact[:12].abs().amax(1)[x[:12].abs().amax(1).double() >= 2.0 ** -113]   # smaller rows: 2^126 does not bring them there
    assert len(m) >= 8
    assert ((m >= 2.0 ** 13) & (m < 2.0 ** 14)).all()
    assert torch.equal(x16[13].isnan(), x[13].isnan()) and x16[14, k - 1] == float("inf") and x16[14].isinf().sum() == 1
    assert x16[15].any() and x16[11].any()
