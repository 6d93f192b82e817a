"""4-bit weights whose scale words pass 2^31 bytes: 2^20 rows of 16384 values in groups of 32, few rows, many and transposed."""
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


def held(got, want, slack):
    got, half = got.double(), HALF_STEP[got.dtype]
    assert ((got - want).abs() <= slack + half * (want.abs() + slack)).all()


def test_scale_words_past_31_bits():
    n, k, group = 1 << 20, 16384, 32
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    codes = torch.empty((n, k), dtype=torch.uint8, device=DEV)
    for a in range(0, n, 1 << 17):
        codes[a:a + (1 << 17)] = torch.randint(0, 16, (1 << 17, k), dtype=torch.uint8, device=DEV, generator=g)
    scales = torch.empty((n, k // group), dtype=torch.float16, device=DEV).normal_(0, 0.01, generator=g)
    zeros = torch.randint(0, 16, (n, k // group), dtype=torch.uint8, device=DEV, generator=g)
    w, ws = ops.w4_pack(codes, scales, zeros, group=group)
    assert ws.nbytes == 1 << 31
    at = torch.arange(k, device=DEV) // group

    def rows_of(r, sign=-1):
        return scales[r].double().abs()[:, at] * (codes[r].double() + zeros[r].double()[:, at]) if sign > 0 else \
            scales[r].double()[:, at] * (codes[r].double() - zeros[r].double()[:, at])

    parts = [slice(0, 40), slice(n // 2 - 20, n // 2 + 20), slice(n - 40, n)]
    for rows, dtype, loss in ((2, torch.float32, 8 * U), (70, torch.bfloat16, 2.0 ** -11)):   # few rows, tiles
        x = torch.empty((rows, k), dtype=dtype, device=DEV).normal_(0, 1, generator=g)
        y = ops.w4_mm(x, w, ws, n, k, group, out_dtype=torch.float32 if rows == 2 else torch.bfloat16)
        for r in parts:
            held(y[:, r], torch.mm(x.double(), rows_of(r).t().contiguous()), (k * U + loss) * torch.mm(x.double().abs(), rows_of(r, 1).t().contiguous()))
    dy = torch.zeros((66, n), dtype=torch.bfloat16, device=DEV)
    for r in parts:
        dy[:, r] = torch.empty((66, 40), device=DEV).normal_(0, 1, generator=g).bfloat16()
    dx = ops.w4_mm_t(dy, w, ws, n, k, group)
    dd, wd = torch.cat([dy[:, r] for r in parts], 1).double(), torch.cat([rows_of(r) for r in parts])
    held(dx, torch.mm(dd, wd), (120 * U + 2.0 ** -11) * torch.mm(dd.abs(), wd.abs()) + 1e-6)
