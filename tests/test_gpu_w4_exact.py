"""Any number of f32 and bf16 rows times 4-bit weights by exact products: the few-row kernel's bound, (K + 8) f32 roundings of the terms
s x q and s x z, where the GEMM behind the same call without `exact` rounds rows and weights to f16."""
import pytest
import torch

from qmm import ops
from ragged_case import U, Guarded, by_expert, gen, held, offsets_of, w4_raw
from test_gpu_w4 import ROW, packed

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("rows,n,k,group,out", [(64, 40, 256, 32, "f32"), (65, 130, 1056, 128, "bf16"), (100, 33, 4096, 64, "f32"), (500, 4200, 160, 128, "f32"),
                                                (333, 8227, 96, 32, "f32"), (1000, 24, 288, ROW, "f32"), (1, 40, 256, 32, "f32"), (0, 40, 256, 32, "f32")])
@pytest.mark.parametrize("x_type", ["f32", "bf16"])
def test_dense(dev, rows, n, k, group, out, x_type):
    g = gen(rows + n)
    raw = w4_raw(g, n, k, group)
    w, ws = packed(raw, group, dev)
    x = torch.randn((rows, k), generator=g).to(T[x_type])
    y = Guarded((rows, n), T[out], dev)
    ops.w4_mm(x.to(dev), w, ws, n, k, group, y=y.t, exact=True)
    y.check()
    held(y.t, x.double() @ raw[3].t(), (k + 8) * U * (x.double().abs() @ raw[4].t()), "exact")


@pytest.mark.parametrize("counts,first,tail,n,k,group", [([300, 0, 200], 2, 3, 40, 256, 32), ([0, 1000, 1], 0, 1, 136, 160, 64), ([70] * 9, 1, 0, 600, 96, 128)])
@pytest.mark.parametrize("x_type", ["f32", "bf16"])
def test_by_expert(dev, counts, first, tail, n, k, group, x_type):
    rows, E, g = first + sum(counts) + tail, len(counts), gen(n)
    offsets = offsets_of(counts, first)
    raw = w4_raw(g, n, k, group, True, E)
    w, ws = packed(raw, group, dev)
    x = torch.randn((rows, k), generator=g).to(T[x_type])
    x[:first], x[rows - tail:] = float("nan"), float("nan")
    y = Guarded((rows, n), torch.float32, dev)
    ops.w4_mm(x.to(dev), w, ws, n, k, group, offsets=offsets.to(dev), y=y.t, exact=True)
    y.check(kept=((0, first), (rows - tail, rows)))
    live = slice(first, rows - tail)
    held(y.t[live], by_expert(x.double(), raw[3], offsets)[live], (k + 8) * U * by_expert(x.double().abs(), raw[4], offsets)[live], "exact by expert")


def test_more_chunks_of_rows_than_a_grid_has(dev):
    """Past 65535 chunks of 64 rows a workgroup takes several."""
    rows, n, k, g = 65535 * 64 + 100, 16, 32, gen(1)
    raw = w4_raw(g, n, k, 32)
    w, ws = packed(raw, 32, dev)
    x = torch.randn((rows, k), generator=g)
    y = ops.w4_mm(x.to(dev), w, ws, n, k, 32, exact=True)
    for part in (slice(0, 200), slice(rows - 300, rows)):
        held(y[part], x[part].double() @ raw[3].t(), (k + 8) * U * (x[part].double().abs() @ raw[4].t()), "many chunks")


def test_graph(dev):
    rows, n, k, g = 100, 40, 512, gen(2)
    w, ws = packed(w4_raw(g, n, k, 64), 64, dev)
    x = torch.randn((rows, k), generator=g).to(dev)
    want = ops.w4_mm(x, w, ws, n, k, 64, exact=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.w4_mm(x, w, ws, n, k, 64, exact=True)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(ops.w4_mm(x, w, ws, n, k, 64, exact=True), want)
