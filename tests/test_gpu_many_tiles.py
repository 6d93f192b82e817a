"""Products of more tiles than a grid's dimension takes: 1024 experts of a row each and matrices 2^20 wide."""
import pytest
import torch

from qmm import ops
from ragged_case import HALF_STEP, U

pytestmark = pytest.mark.gpu
DEV = "cuda"
E, WIDE = 1024, 1 << 20


@pytest.fixture(autouse=True)
def emptied():
    yield
    torch.cuda.empty_cache()


@pytest.fixture
def offsets():
    """Every expert has a row but for two, whose rows a neighbour has, and row 0 and the last belong to none."""
    counts = [1] * E
    counts[5], counts[6], counts[E - 3], counts[E - 2] = 0, 2, 2, 0
    return torch.tensor([1] + counts).cumsum(0)


def normal(shape, scale=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(shape[0] + shape[-1])
    return torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(0, scale, generator=g)


def expert_of(offsets, rows):
    """Row t's expert, None for rows of none."""
    o = offsets.tolist()
    out = [None] * rows
    for e in range(E):
        for t in range(o[e], o[e + 1]):
            out[t] = e
    return out


def check_rows(y, offsets, product, terms, depth):
    """Rows at both ends and between against 64 bits, rows of no expert zero."""
    at = expert_of(offsets, y.shape[0])
    assert not y[0].any() and not y[-1].any() and at[0] is None and at[-1] is None
    for t in (1, 2, 5, 6, 7, 300, 511, 512, 513, 777, E - 3, E - 2, E - 1, E):
        got, want, size = y[t].double(), product(t, at[t]), terms(t, at[t])
        slack = depth * U * size
        assert ((got - want).abs() <= slack + HALF_STEP[y.dtype] * (want.abs() + slack)).all(), t


def test_ragged(offsets):
    rows, narrow = E + 2, 8
    od = offsets.int().to(DEV)
    x, w = normal((rows, narrow)), normal((E, WIDE, narrow))
    y = ops.ragged_mm(x, od, w)
    check_rows(y, offsets, lambda t, e: w[e].double() @ x[t].double(), lambda t, e: w[e].double().abs() @ x[t].double().abs(), narrow)
    wt = w.view(E, narrow, WIDE)
    dx = ops.ragged_mm_t(x, od, wt)
    check_rows(dx, offsets, lambda t, e: x[t].double() @ wt[e].double(), lambda t, e: x[t].double().abs() @ wt[e].double().abs(), narrow)
    del w, wt, y
    dy = dx   # 2^20 wide rows
    dw = ops.ragged_mm_dw(x, dy, od)
    o = offsets.tolist()
    for e in (0, 4, 5, 6, 7, 500, 512, E - 3, E - 2, E - 1):
        a, b = x[o[e]:o[e + 1]].double(), dy[o[e]:o[e + 1]].double()
        want, slack = a.t() @ b, 2 * U * (a.abs().t() @ b.abs())
        assert ((dw[e].double() - want).abs() <= slack + HALF_STEP[dw.dtype] * (want.abs() + slack)).all(), e


def test_four_bit(offsets):
    rows, n, group = E + 2, 8, 1 << 20
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    od = offsets.int().to(DEV)
    codes = torch.randint(0, 16, (E, n, WIDE), dtype=torch.uint8, device=DEV, generator=g)
    scales = torch.empty((E, n, 1), dtype=torch.float16, device=DEV).normal_(0, 0.01, generator=g)
    w, ws = ops.w4_pack(codes, scales, group=group)
    dy = normal((rows, n))
    dx = ops.w4_mm_t(dy, w, ws, n, WIDE, group, offsets=od, out_dtype=torch.bfloat16)
    value = lambda e: scales[e].double() * (codes[e].double() - 8)
    check_rows(dx, offsets, lambda t, e: dy[t].double() @ value(e), lambda t, e: dy[t].double().abs() @ value(e).abs() * (1 + 2.0 ** -11 / (8 * U)), n)


def test_wide_outputs():
    """The 4-bit forward product of one expert 2^20 wide for each of 600 rows through the GEMM."""
    experts, k, group, rows = 600, 32, 32, 602
    g = torch.Generator(device=DEV)
    g.manual_seed(4)
    codes = torch.randint(0, 16, (experts, WIDE, k), dtype=torch.uint8, device=DEV, generator=g)
    scales = torch.empty((experts, WIDE, 1), dtype=torch.float16, device=DEV).normal_(0, 0.01, generator=g)
    w, ws = ops.w4_pack(codes, scales, group=group)
    x = normal((rows, k)).half()
    od = (torch.arange(experts + 1) + 1).int().to(DEV)
    y = ops.w4_mm(x, w, ws, WIDE, k, group, offsets=od, out_dtype=torch.bfloat16)
    assert not y[0].any() and not y[-1].any()
    for t in (1, 2, 255, 256, 512, 513, 600):
        v = scales[t - 1].double() * (codes[t - 1].double() - 8)
        want, size = v @ x[t].double(), v.abs() @ x[t].double().abs()
        slack = (2.0 ** -11 + k * U) * size
        assert ((y[t].double() - want).abs() <= slack + HALF_STEP[y.dtype] * (want.abs() + slack)).all(), t
