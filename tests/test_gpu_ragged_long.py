"""4-bit and ragged products on tensors past 2^32 bytes and 2^31 values: weights of a late expert, late rows of the inputs and the
outputs. Parts of the outputs against 64 bits."""
import pytest
import torch

from qmm import ops
from ragged_case import HALF_STEP, U

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def emptied():
    yield
    torch.cuda.empty_cache()


def normal(shape, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(sum(shape))
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0, scale, generator=g)


def held(got, want, slack):
    got = got.double()
    lim = slack + HALF_STEP[torch.bfloat16] * (want.abs() + slack)   # outputs are bf16 here, f32 ones well inside
    assert ((got - want).abs() <= lim).all(), float(((got - want).abs() / lim).max())


def test_late_experts(dev):
    """600 experts of 8 MB each: the first and the last, by the few-row kernel, by tiles and transposed."""
    E, n, k = 600, 2048, 2048
    w = normal((E, n, k))
    for rows, first in ((20, 7), (500, 200)):
        offsets = torch.tensor([0] + [first] * (E - 1) + [rows], dtype=torch.int32, device=DEV)
        x, dy = normal((rows, k)), normal((rows, n))
        y, dx = ops.ragged_mm(x, offsets, w, out_dtype=torch.float32), ops.ragged_mm_t(dy, offsets, w, out_dtype=torch.float32)
        dw = ops.ragged_mm_dw(dy, x, offsets)
        for e, part in ((0, slice(0, first)), (E - 1, slice(first, rows))):
            xd, dd, wd = x[part].double(), dy[part].double(), w[e].double()
            held(y[part], torch.mm(xd, wd.t().contiguous()), k * U * torch.mm(xd.abs(), wd.abs().t().contiguous()))
            held(dx[part], torch.mm(dd, wd), n * U * torch.mm(dd.abs(), wd.abs()))
            held(dw[e], torch.mm(dd.t().contiguous(), xd), rows * U * torch.mm(dd.abs().t().contiguous(), xd.abs()))
        assert not dw[1:E - 1].any()


def test_wide_matrices(dev):
    """Two experts of 5.4 GB each."""
    E, n, k, rows = 2, 40960, 65536, 75
    w = normal((E, n, k), scale=0.01)
    offsets = torch.tensor([0, 5, rows], dtype=torch.int32, device=DEV)
    x, dy = normal((rows, k)), normal((rows, n))
    y, dx = ops.ragged_mm(x, offsets, w), ops.ragged_mm_t(dy, offsets, w)
    for e, part in ((0, slice(0, 5)), (1, slice(5, rows))):
        for c in (slice(0, 70), slice(n - 70, n)):
            xd, wd = x[part].double(), w[e, c].double().t().contiguous()
            held(y[part, c], torch.mm(xd, wd), k * U * torch.mm(xd.abs(), wd.abs()))
        for c in (slice(0, 70), slice(k - 70, k)):
            dd, wd = dy[part].double(), w[e, :, c].double()
            held(dx[part, c], torch.mm(dd, wd), n * U * torch.mm(dd.abs(), wd.abs()))


def test_many_rows(dev):
    """4.2 million rows of 520 values into as many: x, y and dy of 4.4 GB and 2.2e9 values each."""
    rows, n, k = (1 << 22) + 37, 520, 520
    offsets = torch.tensor([0, 100, 100, rows - 5], dtype=torch.int32, device=DEV)
    x, w = normal((rows, k)), normal((3, n, k), scale=0.05)
    y = torch.full((rows, n), 3.0, dtype=torch.bfloat16, device=DEV)
    ops.ragged_mm(x, offsets, w, y=y)
    late = slice(rows - 305, rows - 5)
    for e, part in ((0, slice(0, 100)), (2, slice(100, 400)), (2, late)):
        xd, wd = x[part].double(), w[e].double().t().contiguous()
        held(y[part], torch.mm(xd, wd), k * U * torch.mm(xd.abs(), wd.abs()))
    assert (y[rows - 5:] == 3).all()
    ops.ragged_mm_t(x, offsets, w, dx=y)
    xd, wd = x[late].double(), w[2].double()
    held(y[late], torch.mm(xd, wd), n * U * torch.mm(xd.abs(), wd.abs()))
    # dW: the late rows alone are not zero
    x[100:rows - 305] = 0
    dw = ops.ragged_mm_dw(y, x, offsets, out_dtype=torch.float32)
    dd, xd = y[late].double(), x[late].double()
    held(dw[2], torch.mm(dd.t().contiguous(), xd), 305 * U * torch.mm(dd.abs().t().contiguous(), xd.abs()))
    assert not dw[1].any()


def test_long_four_bit_weights(dev):
    """One packed matrix of 5.1 GB, few rows, many and transposed; and many rows of a small one."""
    n, k, group = 1 << 17, 80000, 128
    groups = -(-k // group)
    codes = torch.empty((n, k), dtype=torch.uint8, device=DEV)
    for a in range(0, n, 1 << 14):
        codes[a:a + (1 << 14)] = torch.randint(0, 16, (1 << 14, k), dtype=torch.uint8, device=DEV)
    scales, zeros = normal((n, groups), torch.float16, 0.01), torch.randint(0, 16, (n, groups), dtype=torch.uint8, device=DEV)
    w, ws = ops.w4_pack(codes, scales, zeros, group=group)
    at = torch.arange(k, device=DEV) // group
    rows_of = lambda r: scales[r].double()[:, at] * (codes[r].double() - zeros[r].double()[:, at])
    x = normal((70, k))
    for rows, out, loss in ((3, torch.float32, 8 * U), (70, torch.bfloat16, 2.0 ** -11)):
        y = ops.w4_mm(x[:rows], w, ws, n, k, group, out_dtype=out)
        for r in (slice(0, 40), slice(n - 40, n)):
            xd, wd = x[:rows].double(), rows_of(r).t().contiguous()
            size = torch.mm(xd.abs(), (scales[r].double().abs()[:, at] * (codes[r].double() + zeros[r].double()[:, at])).t().contiguous())
            held(y[:, r], torch.mm(xd, wd), (k * U + loss) * size)
    dy = torch.zeros((66, n), device=DEV, dtype=torch.bfloat16)
    dy[:, :50], dy[:, n - 50:] = normal((66, 50)), normal((66, 50))
    dx = ops.w4_mm_t(dy, w, ws, n, k, group)
    dd = torch.cat([dy[:, :50], dy[:, n - 50:]], 1).double()
    wd = torch.cat([rows_of(slice(0, 50)), rows_of(slice(n - 50, n))])
    held(dx, torch.mm(dd, wd), (100 * U + 2.0 ** -11) * torch.mm(dd.abs(), wd.abs()) + 1e-6)
    del codes, w, ws, y, dx
    torch.cuda.empty_cache()
    rows, n, k = (1 << 22) + 37, 544, 544
    codes, scales = torch.randint(0, 16, (n, k), dtype=torch.uint8, device=DEV), normal((n, 5), torch.float16, 0.01)
    w, ws = ops.w4_pack(codes, scales, group=128)
    wd = (scales.double()[:, torch.arange(k, device=DEV) // 128] * (codes.double() - 8)).t().contiguous()
    x = normal((rows, k))
    y = ops.w4_mm(x, w, ws, n, k, 128, out_dtype=torch.bfloat16)
    for part in (slice(0, 300), slice(rows - 300, rows)):
        xd = x[part].double()
        held(y[part], torch.mm(xd, wd), (k * U + 2.0 ** -11) * torch.mm(xd.abs(), wd.abs()) + 1e-6)
    y = ops.w4_mm_t(x, w, ws, n, k, 128, out_dtype=torch.bfloat16)
    xd, wt = x[-300:].double(), wd.t().contiguous()
    held(y[-300:], torch.mm(xd, wt), (n * U + 2.0 ** -11) * torch.mm(xd.abs(), wt.abs()) + 1e-6)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,k", [(1032, 2080), (1000, 4160)])   # whole lines a row in f32 (or both types), part of a tile's columns, rows
def test_weight_gradients_past_the_cache(dev, out, n, k):
    """Outputs past 256 MB: those of whole 128-byte lines a row are stored past the cache, at any other address as elsewhere."""
    counts = [70, 0, 3, 130, 64, 1] * 12
    E, rows = len(counts), sum(counts)
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    x, dy = normal((rows, k)), normal((rows, n))
    buf = torch.full((E * n * k + 512,), 3.0, dtype=out, device=DEV)
    for first in (256, 264):   # 128-byte lines, and not
        dw = buf[first:first + E * n * k].view(E, n, k)
        assert dw.nbytes > 256 << 20
        ops.ragged_mm_dw(dy, x, offsets.to(DEV), dw=dw)
        for e in (0, 1, 2, 3, E - 1):
            a, b = int(offsets[e]), int(offsets[e + 1])
            dd, xd = dy[a:b].double().t().contiguous(), x[a:b].double()
            held(dw[e], torch.mm(dd, xd), 130 * U * torch.mm(dd.abs(), xd.abs()))
        assert not dw[1::6].any()
        assert (buf[:first] == 3).all() and (buf[first + E * n * k:] == 3).all()
        buf.fill_(3.0)
