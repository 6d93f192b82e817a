"""Every kernel of the 4-bit and ragged products against 64 bits: each tile with each group of scales or type, whole sums and sums in
parts (tests/tile_cases.py; test_tile_plans.py holds the cases to their tiles), and each form of the few-row kernel."""
import pytest
import torch

from qmm import ops
from ragged_case import U, Guarded, by_expert, gen, held, offsets_of, spans, w4_raw
from test_gpu_w4 import ROW, packed
from tile_cases import RAGGED, RAGGED_DW, RAGGED_T, W4, W4_T, of, rows_of

pytestmark = pytest.mark.gpu
HALF = [torch.bfloat16, torch.float16]
# ragged_case.held counts half a step of an output relative to its value; below 2^-14 f16's step is 2^-24 whatever the value, and a rounding
# off by half of it
STEP = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
GROUPS = [32, 64, 128, ROW]


def four_bit(dev, counts, first, tail, n, k, group):
    E, g = len(counts), gen(n + k + sum(counts))
    raw = w4_raw(g, n, k, group, True, E)
    return packed(raw, group, dev), raw[3].to(dev), offsets_of(counts, first).to(dev), g


@pytest.mark.parametrize("counts,first,tail,n,k,tile", of(W4))
@pytest.mark.parametrize("group", GROUPS)
def test_four_bit(dev, counts, first, tail, n, k, tile, group):
    rows = rows_of(counts, first, tail)
    (w, ws), wd, offsets, g = four_bit(dev, counts, first, tail, n, k, group)
    x16, scales = ops.row_scale_f16(torch.randn((rows, k), generator=g).to(dev))
    x16[:first], x16[rows - tail:] = float("nan"), float("inf")
    y = Guarded((rows, n), torch.float32, dev)
    ops.w4_mm(x16, w, ws, n, k, group, offsets=offsets, scales=scales, y=y.t)
    y.check(kept=((0, first), (rows - tail, rows)))
    live, xd = slice(first, rows - tail), x16.double() * scales.double()[:, 1:]
    held(y.t[live], by_expert(xd, wd, offsets)[live].cpu(), ((2.0 ** -11 + k * U) * by_expert(xd.abs(), wd.abs(), offsets))[live].cpu(), str(tile))


@pytest.mark.parametrize("counts,first,tail,n,k,tile", of(W4_T))
@pytest.mark.parametrize("group", GROUPS)
def test_four_bit_transposed(dev, counts, first, tail, n, k, tile, group):
    rows = rows_of(counts, first, tail)
    (w, ws), wd, offsets, g = four_bit(dev, counts, first, tail, n, k, group)
    dy = torch.randn((rows, n), generator=g).bfloat16().to(dev)
    y = Guarded((rows, k), torch.float32, dev)
    ops.w4_mm_t(dy, w, ws, n, k, group, offsets=offsets, y=y.t)
    y.check(kept=((0, first), (rows - tail, rows)))
    live, dd = slice(first, rows - tail), dy.double()
    lost = 2.0 ** -38 * dd.abs().amax(-1, keepdim=True).cpu() * by_expert(torch.ones_like(dd), wd.abs(), offsets, t=True)
    slack = (2.0 ** -11 + n * U) * by_expert(dd.abs(), wd.abs(), offsets, t=True) + lost
    held(y.t[live], by_expert(dd, wd, offsets, t=True)[live].cpu(), slack[live].cpu(), str(tile))


def ragged_inputs(dev, counts, first, tail, n, k, dtype):
    rows, E = rows_of(counts, first, tail), len(counts)
    g = torch.Generator(device=dev)
    g.manual_seed(rows + n + k)
    x, dy, w = (torch.randn(s, generator=g, device=dev).to(dtype) for s in ((rows, k), (rows, n), (E, n, k)))
    x[:first], dy[:first], x[rows - tail:], dy[rows - tail:] = (float("nan"),) * 4
    return rows, x, dy, w, offsets_of(counts, first).to(dev)


@pytest.mark.parametrize("counts,first,tail,n,k,tile", of(RAGGED))
@pytest.mark.parametrize("dtype", HALF)
def test_ragged(dev, counts, first, tail, n, k, tile, dtype):
    rows, x, _, w, offsets = ragged_inputs(dev, counts, first, tail, n, k, dtype)
    live = slice(first, rows - tail)
    want, size = by_expert(x.double(), w.double(), offsets)[live].cpu(), by_expert(x.double().abs(), w.double().abs(), offsets)[live].cpu()
    for out in (torch.float32, dtype):
        y = Guarded((rows, n), out, dev)
        ops.ragged_mm(x, offsets, w, y=y.t)
        y.check(kept=((0, first), (rows - tail, rows)))
        held(y.t[live], want, k * U * size + STEP[out], str(tile))


@pytest.mark.parametrize("counts,first,tail,n,k,tile", of(RAGGED_T))
@pytest.mark.parametrize("dtype", HALF)
def test_ragged_transposed(dev, counts, first, tail, n, k, tile, dtype):
    rows, _, dy, w, offsets = ragged_inputs(dev, counts, first, tail, n, k, dtype)
    live = slice(first, rows - tail)
    want, size = by_expert(dy.double(), w.double(), offsets, t=True)[live].cpu(), by_expert(dy.double().abs(), w.double().abs(), offsets, t=True)[live].cpu()
    for out in (torch.float32, dtype):
        dx = Guarded((rows, k), out, dev)
        ops.ragged_mm_t(dy, offsets, w, dx=dx.t)
        dx.check(kept=((0, first), (rows - tail, rows)))
        held(dx.t[live], want, n * U * size + STEP[out], str(tile))


@pytest.mark.parametrize("counts,first,tail,n,k,tile", of(RAGGED_DW))
@pytest.mark.parametrize("dtype", HALF)
def test_weight_gradient(dev, counts, first, tail, n, k, tile, dtype):
    rows, x, dy, _, offsets = ragged_inputs(dev, counts, first, tail, n, k, dtype)
    x, dy = x * 0.125, dy * 0.125   # sums of f16 results stay finite
    for out in (torch.float32, dtype):
        dw = Guarded((len(counts), n, k), out, dev)
        ops.ragged_mm_dw(dy, x, offsets, dw=dw.t)
        dw.check()
        for e, (a, b) in enumerate(spans(offsets.cpu(), rows)):
            xd, dd = x[a:b].double(), dy[a:b].double().t().contiguous()
            held(dw.t[e], torch.mm(dd, xd).cpu(), (b - a) * U * torch.mm(dd.abs(), xd.abs()).cpu() + STEP[out], f"{tile} expert {e}")


# one, two and three row blocks a wave (up to 256, up to 512 and more blocks of 16 rows), one, two and four tiles of 16 tokens; one row
@pytest.mark.parametrize("rows", [1, 9, 20, 40])
@pytest.mark.parametrize("n", [130, 4201, 8260])
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("x_type", [torch.bfloat16, torch.float32])
def test_few_rows(dev, rows, n, group, x_type):
    k, g = 288, gen(rows + n)
    raw = w4_raw(g, n, k, group)
    w, ws = packed(raw, group, dev)
    x = torch.randn((rows, k), generator=g).to(x_type)
    y = Guarded((rows, n), torch.float32, dev)
    ops.w4_mm(x.to(dev), w, ws, n, k, group, y=y.t)
    y.check()
    held(y.t, x.double() @ raw[3].t(), (k + 8) * U * (x.double().abs() @ raw[4].t()), "few rows")


# a row an expert at most on average: waves of their own row blocks where those are 2048 and more, the kernel of several rows below
@pytest.mark.parametrize("E,n", [(256, 140), (30, 90)])
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("x_type", [torch.bfloat16, torch.float32])
def test_a_row_an_expert(dev, E, n, group, x_type):
    k, g = 416, gen(E + n)
    counts = [(1, 0, 1, 2, 1, 0, 1, 1)[i % 8] for i in range(E)]
    counts[-1] += E - sum(counts) - 1
    offsets = offsets_of(counts, 1)
    rows = E
    raw = w4_raw(g, n, k, group, True, E)
    w, ws = packed(raw, group, dev)
    x = torch.randn((rows, k), generator=g).to(x_type)
    x[0] = float("nan")
    y = Guarded((rows, n), torch.float32, dev)
    ops.w4_mm(x.to(dev), w, ws, n, k, group, offsets=offsets.to(dev), y=y.t)
    y.check(kept=((0, 1),))
    held(y.t[1:], by_expert(x.double(), raw[3], offsets)[1:], (k + 8) * U * by_expert(x.double().abs(), raw[4], offsets)[1:], "a row an expert")


@pytest.mark.parametrize("counts", [[1], [1, 0, 1, 1, 0, 2, 0, 0], [12], [20], [5, 0, 40], [64]])
@pytest.mark.parametrize("dtype", HALF)
def test_few_rows_of_16_bits(dev, counts, dtype):
    n, k, rows, E = 136, 520, sum(counts), len(counts)
    g, offsets = gen(rows), offsets_of(counts)
    x, w = torch.randn((rows, k), generator=g).to(dtype), torch.randn((E, n, k), generator=g).to(dtype)
    for out in (torch.float32, dtype):
        y = Guarded((rows, n), out, dev)
        ops.ragged_mm(x.to(dev), offsets.to(dev), w.to(dev), y=y.t)
        y.check()
        held(y.t, by_expert(x.double(), w.double(), offsets), k * U * by_expert(x.double().abs(), w.double().abs(), offsets) + STEP[out], "few rows")


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("rows,n,k", [(70, 40, 160), (300, 264, 288)])
def test_small_scales(dev, rows, n, k, group):
    """Scales among f16's subnormals: weights s (q - z) are multiples of 2^-24 below 2^-13 and enter exactly, in tiles both ways."""
    g = gen(rows)
    q, _, z, _, _ = w4_raw(g, n, k, group)
    s = torch.randint(-40, 41, (n, -(-k // group)), generator=g).double().mul(2.0 ** -24).half()
    at = torch.arange(k) // group
    wd = s.double()[:, at] * (q.double() - z.double()[:, at])
    assert torch.equal(wd.half().double(), wd) and 0 < float(wd.abs().max()) < 2.0 ** -13
    w, ws = packed((q, s, z), group, dev)
    x, dy = torch.randint(-8, 9, (rows, k), generator=g).bfloat16(), torch.randint(-8, 9, (rows, n), generator=g).bfloat16()
    y = ops.w4_mm(x.to(dev), w, ws, n, k, group)
    dx = ops.w4_mm_t(dy.to(dev), w, ws, n, k, group)
    # small integers times multiples of 2^-24: every sum is exact
    assert torch.equal(y.cpu().double(), x.double() @ wd.t()) and torch.equal(dx.cpu().double(), dy.double() @ wd)
