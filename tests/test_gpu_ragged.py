"""Ragged products of 16-bit expert weights and their gradients against 64 bits: empty experts, one row, segments that end inside
a tile, rows of no expert before and behind, columns that end inside a tile."""
import pytest
import torch

from qmm import ops
from ragged_case import U, Guarded, by_expert, gen, held, offsets_of, spans

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CASES = [  # counts, rows before, rows behind, n, k, type, output
    ([1], 0, 0, 8, 8, "bf16", "f32"),
    ([0, 2, 0, 1], 0, 0, 24, 40, "bf16", "bf16"),
    ([3, 16, 17, 0], 2, 1, 136, 264, "f16", "f32"),
    ([1] * 40 + [0] * 60 + [2], 0, 0, 16, 96, "bf16", "f32"),
    ([64, 65, 1, 0], 0, 3, 72, 128, "bf16", "bf16"),
    ([129, 0, 0, 127], 5, 0, 200, 392, "f16", "f16"),
    ([0, 0, 0], 0, 2, 16, 16, "bf16", "f32"),
    ([300, 520], 0, 0, 264, 136, "bf16", "f32"),
    ([0, 700, 1, 90], 1, 7, 520, 328, "bf16", "bf16"),
    ([200] * 5, 0, 0, 384, 512, "f16", "f32"),
    # thousands of rows
    ([30, 0, 31, 90, 1, 28] * 17, 3, 2, 600, 616, "bf16", "f32"),
    ([1100, 0, 903], 0, 0, 1032, 520, "bf16", "bf16"),
    ([4000, 4101], 0, 5, 1000, 200, "f16", "f32"),
    ([8000, 1, 0, 8300], 2, 0, 1000, 136, "bf16", "bf16"),
    # long sums of few outputs in parts: the forward, the input's gradient, the weights'
    ([640, 0, 300], 3, 5, 72, 16384, "bf16", "bf16"),
    ([100, 0, 61], 2, 1, 8200, 64, "f16", "f32"),
    ([7000, 0, 3], 0, 4, 64, 72, "bf16", "bf16"),
]


def inputs(counts, first, tail, n, k, dtype):
    rows = first + sum(counts) + tail
    g = gen(rows + n + k)
    x = torch.randn((rows, k), generator=g).to(T[dtype])
    dy = (torch.randn((rows, n), generator=g) * 0.1).to(T[dtype])
    w = torch.randn((len(counts), n, k), generator=g).div(k ** 0.5).to(T[dtype])
    x[:first], dy[:first], x[rows - tail:], dy[rows - tail:] = (float("nan"),) * 4   # rows of no expert are not read into anything
    return rows, x, dy, w, offsets_of(counts, first)


@pytest.mark.parametrize("counts,first,tail,n,k,dtype,out", CASES)
def test_forward(dev, counts, first, tail, n, k, dtype, out):
    rows, x, _, w, offsets = inputs(counts, first, tail, n, k, dtype)
    y = Guarded((rows, n), T[out], dev)
    ops.ragged_mm(x.to(dev), offsets.to(dev), w.to(dev), y=y.t)
    y.check(kept=((0, first), (rows - tail, rows)))
    live = slice(first, rows - tail)
    held(y.t[live], by_expert(x.double(), w.double(), offsets)[live], (k * U * by_expert(x.double().abs(), w.double().abs(), offsets))[live], "ragged")


@pytest.mark.parametrize("counts,first,tail,n,k,dtype,out", CASES)
def test_input_gradient(dev, counts, first, tail, n, k, dtype, out):
    rows, _, dy, w, offsets = inputs(counts, first, tail, n, k, dtype)
    dx = Guarded((rows, k), T[out], dev)
    ops.ragged_mm_t(dy.to(dev), offsets.to(dev), w.to(dev), dx=dx.t)
    dx.check(kept=((0, first), (rows - tail, rows)))
    live = slice(first, rows - tail)
    held(dx.t[live], by_expert(dy.double(), w.double(), offsets, t=True)[live],
         (n * U * by_expert(dy.double().abs(), w.double().abs(), offsets, t=True))[live], "ragged dx")


@pytest.mark.parametrize("counts,first,tail,n,k,dtype,out", CASES)
def test_weight_gradient(dev, counts, first, tail, n, k, dtype, out):
    rows, x, dy, w, offsets = inputs(counts, first, tail, n, k, dtype)
    dw = Guarded(tuple(w.shape), T[out], dev)
    ops.ragged_mm_dw(dy.to(dev), x.to(dev), offsets.to(dev), dw=dw.t)
    dw.check()
    xd, dd = x.double(), dy.double()
    want = torch.stack([dd[a:b].t() @ xd[a:b] for a, b in spans(offsets, rows)])
    size = torch.stack([dd[a:b].abs().t() @ xd[a:b].abs() for a, b in spans(offsets, rows)])
    held(dw.t, want, max(max(counts), 1) * U * size, "ragged dw")
    empty = [e for e, c in enumerate(counts) if c == 0]
    assert not dw.t[empty].any()


def test_gradients_against_differences(dev):
    """L = sum dy y(x, w) is linear in x and in w: a difference over a direction is the gradient's product with it."""
    rows, x, dy, w, offsets = inputs([5, 0, 70, 33], 0, 0, 64, 96, "bf16")
    g = gen(4)
    ex, ew = torch.randint(-1, 2, x.shape, generator=g).to(x), torch.randint(-1, 2, w.shape, generator=g).to(w)
    run = lambda a, b: (ops.ragged_mm(a.to(dev), offsets.to(dev), b.to(dev), out_dtype=torch.float32).cpu().double() * dy.double()).sum()
    dx, dw = ops.ragged_mm_backward(dy.to(dev), x.to(dev), offsets.to(dev), w.to(dev), out_dtype=torch.float32, dw_dtype=torch.float32)
    for grad, e, value in ((dx, ex, run(ex, w)), (dw, ew, run(x, ew))):   # linear: L(x + e) - L(x) is L(e)
        want = (grad.cpu().double() * e.double()).sum()
        size = (by_expert((ex if e is ex else x).double().abs(), (w if e is ex else ew).double().abs(), offsets) * dy.double().abs()).sum()
        assert (value - want).abs() <= (96 + 64 + 70) * U * size


def test_no_rows(dev):
    w = torch.randn((3, 16, 24), device=dev).bfloat16()
    offsets = torch.zeros(4, dtype=torch.int32, device=dev)
    x, dy = torch.zeros((0, 24), device=dev).bfloat16(), torch.zeros((0, 16), device=dev).bfloat16()
    assert ops.ragged_mm(x, offsets, w).shape == (0, 16)
    dx, dw = ops.ragged_mm_backward(dy, x, offsets, w)
    assert dx.shape == (0, 24) and dw.shape == (3, 16, 24) and not dw.any()


@pytest.mark.parametrize("rows", [9, 300])
def test_offsets_out_of_range_are_clamped(dev, rows):
    x, dy = torch.randn((rows, 40), generator=gen(1)).bfloat16(), torch.randn((rows, 24), generator=gen(2)).bfloat16()
    w = torch.randn((4, 24, 40), generator=gen(3)).bfloat16()
    offsets = torch.tensor([-3, 5, 1, rows + 9, 2 ** 31 - 1], dtype=torch.int32)   # experts 1 and 3 are empty
    y, dx = Guarded((rows, 24), torch.float32, dev), Guarded((rows, 40), torch.float32, dev)
    ops.ragged_mm(x.to(dev), offsets.to(dev), w.to(dev), y=y.t)
    ops.ragged_mm_t(dy.to(dev), offsets.to(dev), w.to(dev), dx=dx.t)
    dw = ops.ragged_mm_dw(dy.to(dev), x.to(dev), offsets.to(dev), out_dtype=torch.float32)
    y.check(), dx.check()
    held(y.t[5:], x[5:].double() @ w[2].double().t(), 40 * U * (x[5:].double().abs() @ w[2].double().abs().t()))
    held(dx.t[5:], dy[5:].double() @ w[2].double(), 24 * U * (dy[5:].double().abs() @ w[2].double().abs()))
    held(dw[2], dy[1:].double().t() @ x[1:].double(), rows * U * (dy[1:].double().abs().t() @ x[1:].double().abs()))
    assert not dw[1].any() and not dw[3].any()


@pytest.mark.parametrize("rows", [4, 400])
def test_stream_and_graph(dev, rows):
    _, x, dy, w, offsets = inputs([rows // 4, 0, rows - rows // 4], 0, 0, 136, 72, "bf16")
    x, dy, w, offsets = (t.to(dev) for t in (x, dy, w, offsets))
    want = (ops.ragged_mm(x, offsets, w), *ops.ragged_mm_backward(dy, x, offsets, w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = (ops.ragged_mm(x, offsets, w), *ops.ragged_mm_backward(dy, x, offsets, w))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = (ops.ragged_mm(x, offsets, w), *ops.ragged_mm_backward(dy, x, offsets, w))
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
