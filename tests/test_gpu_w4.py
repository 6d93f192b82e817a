"""Products on 4-bit weights with group scales against 64 bits: few rows and many, dense and by expert, both directions, at the
sizes where tiles, groups, rows and columns end inside a unit of work."""
import pytest
import torch

from qmm import ops
from ragged_case import U, Guarded, by_expert, gen, held, offsets_of, spans, w4_raw

pytestmark = pytest.mark.gpu
ROW = 1 << 20   # one scale a row
T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def packed(raw, group, dev):
    q, s, z = raw[:3]
    return ops.w4_pack(q.to(dev), s.to(dev), None if z is None else z.to(dev), group=group)


def layout(q, s, z):
    """The packed words a value at a time."""
    n, k = q.shape
    nt = -(-k // 128)
    w = torch.zeros((-(-n // 16), nt, 64, 4), dtype=torch.int64)
    for r in range(n):
        for c in range(k):
            t, rest = divmod(c, 128)
            j, rest = divmod(rest, 32)
            h, v = divmod(rest, 8)
            w[r // 16, t, 16 * h + r % 16, j] |= int(q[r, c]) << (8 * (v % 4) + 4 * (v // 4))
    words = torch.full((-(-n // 16), s.shape[1], 16), 0x64000000, dtype=torch.int64)
    for r in range(n):
        for g in range(s.shape[1]):
            words[r // 16, g, r % 16] = (int(s[r, g].view(torch.int16)) & 0xFFFF) | (0x6400 + (8 if z is None else int(z[r, g]))) << 16
    return w.reshape(-1), words.reshape(-1)


@pytest.mark.parametrize("n,k,group,zeros", [(1, 32, 32, True), (17, 160, 64, True), (33, 256, 128, False), (16, 128, ROW, True)])
def test_pack(dev, n, k, group, zeros):
    raw = w4_raw(gen(n + k), n, k, group, zeros)
    w, ws = packed(raw, group, dev)
    want, words = layout(*raw[:3])
    assert torch.equal(w.cpu().view(torch.int32).long() & 0xFFFFFFFF, want)
    assert torch.equal(ws.cpu().long() & 0xFFFFFFFF, words)


def few_case(dev, rows, n, k, group, zeros, x_type, out, offsets=None, E=None, seed=0, operand=False):
    g = gen(rows * 1000 + n + k + seed)
    raw = w4_raw(g, n, k, group, zeros, E)
    x = (torch.randn((rows, k), generator=g) * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g).float())).to(T[x_type])
    w, ws = packed(raw, group, dev)
    y = Guarded((rows, n), T[out], dev)
    xd, scales = ops.row_scale_f16(x.to(dev)) if operand and x_type != "f16" else (x.to(dev), None)   # the operand takes the GEMM
    got = ops.w4_mm(xd, w, ws, n, k, group, offsets=None if offsets is None else offsets.to(dev), scales=scales, y=y.t)
    assert got.data_ptr() == y.t.data_ptr()
    return x, raw, y


FEW = [(1, 1, 32, 32, True, "f32", "f32"), (1, 17, 160, 64, True, "bf16", "f32"), (1, 768, 4096, 128, False, "bf16", "bf16"),
       (2, 48, 2048, ROW, True, "f32", "f32"), (3, 100, 288, 32, False, "f32", "bf16"), (5, 64, 1184, 128, True, "f32", "f32"),
       (16, 33, 512, 256, True, "bf16", "f32"), (17, 40, 640, 64, True, "f32", "f32"), (31, 16, 96, 32, True, "bf16", "bf16"),
       (33, 130, 1056, 128, True, "bf16", "f32"), (63, 50, 384, 32, True, "f32", "f32"), (63, 20, 5120, 512, False, "bf16", "f32")]


@pytest.mark.parametrize("rows,n,k,group,zeros,x_type,out", FEW)
def test_few_rows(dev, rows, n, k, group, zeros, x_type, out):
    x, raw, y = few_case(dev, rows, n, k, group, zeros, x_type, out)
    y.check()
    # the terms are s q x and s z x apart (the zero point joins after the sums)
    held(y.t, x.double() @ raw[3].t(), (k + 8) * U * (x.double().abs() @ raw[4].t()), "w4 few rows")


@pytest.mark.parametrize("counts,first,tail,n,k,group,x_type,out", [
    ([1, 0, 3, 0, 0, 2], 0, 0, 40, 256, 128, "bf16", "f32"), ([0, 0, 40, 1], 2, 5, 24, 160, 32, "f32", "f32"),
    ([0, 0, 0], 0, 3, 16, 128, 64, "f32", "f32"), ([2] * 70 + [0] * 60, 1, 0, 16, 96, 32, "bf16", "bf16"),
    ([17, 1, 30], 0, 0, 33, 288, ROW, "f32", "f32")])
def test_few_rows_by_expert(dev, counts, first, tail, n, k, group, x_type, out):
    rows, E = first + sum(counts) + tail, len(counts)
    offsets = offsets_of(counts, first)
    x, raw, y = few_case(dev, rows, n, k, group, True, x_type, out, offsets, E)
    y.check(kept=((0, first), (rows - tail, rows)))
    live = slice(first, rows - tail)
    held(y.t[live], by_expert(x.double(), raw[3], offsets)[live], (k + 8) * U * by_expert(x.double().abs(), raw[4], offsets)[live], "w4 few rows by expert")


def row_rounding(x, absw, terms):
    """What row_scale_f16 (and the gradient operand) may lose of the rows x: subnormals, and f32's bits past f16's."""
    lost = 2.0 ** -38 * x.double().abs().amax(-1, keepdim=True) * absw
    return lost + (2.0 ** -11 * terms if x.dtype == torch.float32 else 0)


MANY = [(64, 8, 32, 32, True, "bf16", "bf16"), (65, 200, 96, 32, True, "bf16", "f32"), (100, 129, 288, 64, False, "f32", "f32"),
        (129, 256, 512, 128, True, "bf16", "bf16"), (200, 257, 160, ROW, True, "bf16", "f32"), (257, 520, 1024, 64, True, "bf16", "bf16"),
        (300, 31, 4096, 128, True, "bf16", "f32"), (1, 40, 256, 128, True, "f16", "f32"), (70, 96, 2048, 256, True, "f16", "bf16"),
        # larger sizes (a case of every tile: tile_cases.py)
        (640, 5000, 160, 32, True, "bf16", "bf16"), (8300, 300, 96, 32, True, "bf16", "f32"), (4090, 2000, 288, 64, True, "bf16", "bf16"),
        # long sums of few outputs, in parts
        (90, 72, 8192, 128, True, "bf16", "f32"), (70, 33, 9088, 32, True, "bf16", "bf16"), (200, 300, 2080, 64, True, "bf16", "f32")]


@pytest.mark.parametrize("rows,n,k,group,zeros,x_type,out", MANY)
def test_many_rows(dev, rows, n, k, group, zeros, x_type, out):
    x, raw, y = few_case(dev, rows, n, k, group, zeros, x_type, out, seed=1, operand=True)
    y.check()
    xd, w = x.double(), raw[3]
    terms = xd.abs() @ w.abs().t()
    held(y.t, xd @ w.t(), (2.0 ** -11 + k * U) * terms + row_rounding(x, w.abs().sum(1), terms) * (x_type != "f16"), "w4 many rows")


def test_f16_operand_with_scales(dev):
    g = gen(5)
    raw = w4_raw(g, 72, 320, 64)
    x = torch.randn((90, 320), generator=g) * 1000
    w, ws = packed(raw, 64, dev)
    x16, scales = ops.row_scale_f16(x.to(dev))
    y = ops.w4_mm(x16, w, ws, 72, 320, 64, scales=scales)
    xd = x16.cpu().double() * scales.cpu().double()[:, 1:]
    held(y, xd @ raw[3].t(), (2.0 ** -11 + 320 * U) * (xd.abs() @ raw[3].abs().t()))
    assert torch.equal(y, ops.w4_mm(x.to(dev), w, ws, 72, 320, 64))


BY_EXPERT = [([70, 0, 130, 1], 0, 0, 136, 288, 32, "bf16"), ([0, 300, 5], 3, 9, 40, 512, 128, "f32"),
             ([33] * 9 + [0, 0], 0, 1, 264, 160, 64, "bf16"), ([0, 0, 600, 280], 0, 0, 300, 256, ROW, "bf16"),
             ([500, 0, 1, 1200, 129] * 2, 7, 3, 1000, 160, 32, "bf16"), ([70, 0, 33], 3, 2, 41, 8192, 128, "f32")]


@pytest.mark.parametrize("counts,first,tail,n,k,group,out", BY_EXPERT)
def test_many_rows_by_expert(dev, counts, first, tail, n, k, group, out):
    rows, E = first + sum(counts) + tail, len(counts)
    offsets = offsets_of(counts, first)
    x, raw, y = few_case(dev, rows, n, k, group, True, "bf16", out, offsets, E, seed=2, operand=True)
    y.check(kept=((0, first), (rows - tail, rows)))
    live = slice(first, rows - tail)
    terms = by_expert(x.double().abs(), raw[3].abs(), offsets)
    ones = by_expert(torch.ones_like(x, dtype=torch.float64), raw[3].abs(), offsets)
    slack = (2.0 ** -11 + k * U) * terms + 2.0 ** -38 * x.double().abs().amax(-1, keepdim=True) * ones
    held(y.t[live], by_expert(x.double(), raw[3], offsets)[live], slack[live], "w4 by expert")


GRADS = [(1, 8, 32, 32, True, "bf16", "f32"), (77, 100, 288, 32, True, "bf16", "bf16"), (64, 17, 160, 64, True, "f32", "f32"),
         (129, 200, 512, 128, False, "bf16", "f32"), (200, 64, 1024, ROW, True, "bf16", "bf16"), (257, 320, 96, 64, True, "bf16", "f32"),
         # larger sizes (a case of every tile: tile_cases.py)
         (16300, 72, 1024, 32, True, "bf16", "bf16"), (8100, 200, 992, 64, True, "bf16", "bf16"), (2000, 130, 1024, 128, True, "bf16", "f32"),
         # long sums in parts
         (77, 8200, 96, 32, True, "bf16", "f32"), (130, 3000, 160, 64, True, "f32", "bf16")]


@pytest.mark.parametrize("rows,n,k,group,zeros,dy_type,out", GRADS)
def test_input_gradient(dev, rows, n, k, group, zeros, dy_type, out):
    g = gen(rows + n + k)
    raw = w4_raw(g, n, k, group, zeros)
    dy = (torch.randn((rows, n), generator=g) * 1e-3).to(T[dy_type])
    w, ws = packed(raw, group, dev)
    y = Guarded((rows, k), T[out], dev)
    ops.w4_mm_t(dy.to(dev), w, ws, n, k, group, y=y.t)
    y.check()
    terms = dy.double().abs() @ raw[3].abs()
    held(y.t, dy.double() @ raw[3], (2.0 ** -11 + n * U) * terms + row_rounding(dy, raw[3].abs().sum(0), terms), "w4 gradient")


@pytest.mark.parametrize("counts,first,tail,n,k,group", [([70, 0, 130, 1], 0, 0, 136, 288, 32), ([0, 500, 2], 4, 3, 40, 512, 128),
                                                         ([9] * 12, 0, 0, 72, 160, ROW), ([900, 0, 2100, 1] * 4, 0, 0, 72, 1024, 32), ([70, 0, 33], 4, 3, 6000, 64, 64)])
def test_input_gradient_by_expert(dev, counts, first, tail, n, k, group):
    rows, E = first + sum(counts) + tail, len(counts)
    g = gen(rows + n)
    raw = w4_raw(g, n, k, group, True, E)
    dy = torch.randn((rows, n), generator=g).bfloat16()
    offsets = offsets_of(counts, first)
    w, ws = packed(raw, group, dev)
    y = Guarded((rows, k), torch.float32, dev)
    ops.w4_mm_t(dy.to(dev), w, ws, n, k, group, offsets=offsets.to(dev), y=y.t)
    y.check(kept=((0, first), (rows - tail, rows)))
    live = slice(first, rows - tail)
    terms = by_expert(dy.double().abs(), raw[3].abs(), offsets, t=True)
    ones = by_expert(torch.ones_like(dy, dtype=torch.float64), raw[3].abs(), offsets, t=True)
    slack = (2.0 ** -11 + n * U) * terms + 2.0 ** -38 * dy.double().abs().amax(-1, keepdim=True) * ones
    held(y.t[live], by_expert(dy.double(), raw[3], offsets, t=True)[live], slack[live], "w4 gradient by expert")


def test_input_gradient_against_differences(dev):
    """y is linear in x: (y(x + e) - y(x - e)) / 2 summed with dy is e . dx."""
    g = gen(11)
    n, k, rows = 96, 160, 3
    raw = w4_raw(g, n, k, 32)
    w, ws = packed(raw, 32, dev)
    x, e, dy = (torch.randn((rows, c), generator=g).bfloat16() for c in (k, k, n))
    step = e.float()   # exact sums below: few-row products are exact up to f32 sums
    hi, lo = (ops.w4_mm((x.float() + v * step).to(dev), w, ws, n, k, 32).cpu().double() for v in (1, -1))
    dx = ops.w4_mm_t(dy.to(dev), w, ws, n, k, 32).cpu().double()
    got, want = (dx * step.double()).sum(), ((hi - lo) / 2 * dy.double()).sum()
    size = (dy.double().abs() @ raw[3].abs() * step.double().abs()).sum()
    both = ((x.float().abs() + step.abs()).double() @ raw[4].t() * dy.double().abs()).sum()
    assert (got - want).abs() <= (2.0 ** -11 + n * U) * size + 2 * (k + 8) * U * both + 2.0 ** -24 * both


def test_no_rows_and_zero_gradient(dev):
    raw = w4_raw(gen(1), 24, 64, 32)
    w, ws = packed(raw, 32, dev)
    assert ops.w4_mm(torch.zeros((0, 64), device=dev), w, ws, 24, 64, 32).shape == (0, 24)
    assert ops.w4_mm_t(torch.zeros((0, 24), device=dev), w, ws, 24, 64, 32).shape == (0, 64)
    assert not ops.w4_mm_t(torch.zeros((70, 24), device=dev), w, ws, 24, 64, 32).any()


def test_a_row_does_not_see_its_neighbours(dev):
    """NaN and infinities of one row stay in it, on both sides of the row count that changes the kernel."""
    raw = w4_raw(gen(2), 48, 256, 64)
    w, ws = packed(raw, 64, dev)
    for rows in (5, 40, 80):
        x = torch.randn((rows, 256), generator=gen(rows)).to(dev)
        clean = ops.w4_mm(x, w, ws, 48, 256, 64)
        x[3, 7], x[4, 100] = float("nan"), float("inf")
        y = ops.w4_mm(x, w, ws, 48, 256, 64)
        rest = [r for r in range(rows) if r not in (3, 4)]
        assert torch.equal(y[rest], clean[rest]) and y[3].isnan().all() and not y[4].isfinite().any()


def test_offsets_out_of_range_are_clamped(dev):
    n, k = 24, 128
    raw = w4_raw(gen(3), n, k, 32, True, 4)
    w, ws = packed(raw, 32, dev)
    for rows in (10, 200):
        x = torch.randn((rows, k), generator=gen(rows)).bfloat16()
        offsets = torch.tensor([-7, 4, 2, rows + 50, 2 ** 31 - 1], dtype=torch.int32)
        y = Guarded((rows, n), torch.float32, dev)
        ops.w4_mm(x.to(dev), w, ws, n, k, 32, offsets=offsets.to(dev), y=y.t)
        y.check()
        a = spans(offsets, rows)
        assert a == [(0, 4), (4, 4), (2, rows), (rows, rows)]
        want = x[4:].double() @ raw[3][2].t()
        held(y.t[4:], want, (2.0 ** -10 + k * U) * (x[4:].double().abs() @ raw[4][2].t()) + 1e-9)


@pytest.mark.parametrize("rows", [3, 100])
def test_stream_and_graph(dev, rows):   # f32 rows: the few-row kernel, then row scale and GEMM
    n, k, E = 80, 256, 5
    raw = w4_raw(gen(rows), n, k, 64, True, E)
    w, ws = packed(raw, 64, dev)
    offsets = offsets_of([rows // 3, 0, rows - rows // 3, 0, 0]).to(dev)
    x = torch.randn((rows, k), generator=gen(9)).to(dev)
    dy = torch.randn((rows, n), generator=gen(10)).bfloat16().to(dev)
    want, dwant = ops.w4_mm(x, w, ws, n, k, 64, offsets=offsets), ops.w4_mm_t(dy, w, ws, n, k, 64, offsets=offsets)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.w4_mm(x, w, ws, n, k, 64, offsets=offsets), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = ops.w4_mm(x, w, ws, n, k, 64, offsets=offsets), ops.w4_mm_t(dy, w, ws, n, k, 64, offsets=offsets)
    for i in range(3):
        y.zero_(), dx.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(dx, dwant)
    x.mul_(0.5)
    graph.replay()
    assert torch.equal(y, ops.w4_mm(x, w, ws, n, k, 64, offsets=offsets))
