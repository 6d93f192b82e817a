"""Rows that the offsets give to no expert: zero in an output that the call makes (they have no part in anything, so that is their
value and their gradient), left as they were in a given one. Every kernel that writes such rows' neighbours: few rows, tiles, sums in
parts; offsets with rows before, behind and between the segments. Memory that a call allocates holds NaN beforehand."""
import contextlib

import pytest
import torch

from qmm import ops
from ragged_case import Guarded, gen, offsets_of, w4_raw
from test_gpu_w4 import packed

pytestmark = pytest.mark.gpu
# steps back between segments (no row belongs to two)
BACKWARDS = [3, 9, 9, 0, 2, 2, 2]        # 3 .. 8 and 0 .. 1: none has 2 and 9 on
JUMPS = [40, 60, 10, 25, 25, 35, 30]     # 40 .. 59, 10 .. 24, 25 .. 34: none has 0 - 9, 35 - 39 and 60 on


@contextlib.contextmanager
def nan_memory():
    """New tensors hold NaN (bytes: 255, which is NaN read as f32)."""
    was = torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True)
    try:
        assert torch.empty(8, device="cuda").isnan().all()
        yield
    finally:
        torch.use_deterministic_algorithms(was)


def none_of(offsets, rows):
    """The rows of no expert, one by one from the definition."""
    o = [min(max(v, 0), rows) for v in offsets.tolist()]
    return torch.tensor([not any(a <= t < b for a, b in zip(o, o[1:])) for t in range(rows)], dtype=torch.bool)


def check(new, given, rest):
    """new: an output that the call made; given: the same call's into a tensor of sentinels."""
    given.check()
    assert not new[rest].any(), "rows of no expert"   # NaN is true
    assert (given.t[rest] == given.fill).all()
    assert torch.equal(new[~rest], given.t[~rest]) and new[~rest].isfinite().all()


# rows, offsets, n, k: few rows, few rows in parts, tiles, tiles in parts, one expert, experts without rows, all rows of none
CASES = [(9, offsets_of([2, 0, 3], 3), 24, 64), (12, torch.tensor(BACKWARDS), 40, 96), (31, offsets_of([9, 12], 4), 24, 12288),
         (300, offsets_of([70, 0, 130, 1], 60), 136, 288), (100, torch.tensor(JUMPS), 72, 160), (200, offsets_of([70, 0, 33], 40), 40, 8192),
         (200, offsets_of([90], 0), 8200, 64), (70, offsets_of([60], 10), 16, 32), (80, offsets_of([0, 0, 0], 5), 24, 64), (5, offsets_of([0, 0], 0), 8, 32),
         (1, offsets_of([0, 0], 1), 8, 32), (5000, offsets_of([1, 1200, 0, 64], 2100), 1000, 416)]


@pytest.mark.parametrize("rows,offsets,n,k", CASES)
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_ragged(dev, rows, offsets, n, k, out):
    E, g = len(offsets) - 1, gen(rows + n)
    x, dy, w = (torch.randn(s, generator=g).bfloat16().to(dev) for s in ((rows, k), (rows, n), (E, n, k)))
    rest = none_of(offsets, rows)
    x[rest], dy[rest] = float("nan"), float("nan")
    od = offsets.int().to(dev)
    y, dx = Guarded((rows, n), out, dev), Guarded((rows, k), out, dev)
    ops.ragged_mm(x, od, w, y=y.t)
    ops.ragged_mm_t(dy, od, w, dx=dx.t)
    dw = ops.ragged_mm_dw(dy, x, od, out_dtype=out)
    with nan_memory():
        check(ops.ragged_mm(x, od, w, out_dtype=out), y, rest)
        check(ops.ragged_mm_t(dy, od, w, out_dtype=out), dx, rest)
        both = ops.ragged_mm_backward(dy, x, od, w, out_dtype=out, dw_dtype=out)
    check(both[0], dx, rest)
    assert torch.equal(both[1], dw)


@pytest.mark.parametrize("rows,offsets,n,k", CASES)
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_four_bit(dev, rows, offsets, n, k, out):
    n += 1   # rows that start at any address
    E, g = len(offsets) - 1, gen(rows + n)
    w, ws = packed(w4_raw(g, n, k, 32, True, E), 32, dev)
    x, dy = (torch.randn(s, generator=g).to(dev) for s in ((rows, k), (rows, n)))
    rest = none_of(offsets, rows)
    od = offsets.int().to(dev)
    y, y16, dx = Guarded((rows, n), out, dev), Guarded((rows, n), out, dev), Guarded((rows, k), out, dev)
    x16, scales = ops.row_scale_f16(x)
    ops.w4_mm(x, w, ws, n, k, 32, offsets=od, y=y.t)
    ops.w4_mm(x16, w, ws, n, k, 32, offsets=od, scales=scales, y=y16.t)
    ops.w4_mm_t(dy, w, ws, n, k, 32, offsets=od, y=dx.t)
    with nan_memory():
        check(ops.w4_mm(x, w, ws, n, k, 32, offsets=od, out_dtype=out), y, rest)
        check(ops.w4_mm(x16, w, ws, n, k, 32, offsets=od, scales=scales, out_dtype=out), y16, rest)
        check(ops.w4_mm_t(dy, w, ws, n, k, 32, offsets=od, out_dtype=out), dx, rest)


def test_a_layer_with_padding_rows(dev):
    """A padded batch: the gradient that a layer adds to its tokens from all rows, those of no expert among them."""
    T, H, F, E, g = 40, 64, 96, 3, gen(1)
    x, w, dy = torch.randn((T, H), generator=g).bfloat16(), torch.randn((E, F, H), generator=g).bfloat16(), torch.randn((T, F), generator=g).bfloat16()
    offsets = offsets_of([8, 0, 20], 5).to(dev)
    tokens = torch.randperm(T, generator=g).to(dev)
    with nan_memory():
        dxs, _ = ops.ragged_mm_backward(dy.to(dev), x.to(dev), offsets, w.to(dev), out_dtype=torch.float32)
    dx = torch.zeros((T, H), device=dev).index_add_(0, tokens, dxs)
    assert dx.isfinite().all() and not dx[tokens[:5]].any() and not dx[tokens[33:]].any() and dx[tokens[5:33]].any(1).all()


@pytest.mark.parametrize("rows", [12, 200])
def test_replayed_with_other_offsets(dev, rows):
    """A captured call's output follows the offsets of each replay."""
    E, n, k, g = 3, 24, 64, gen(rows)
    x, w = torch.randn((rows, k), generator=g).bfloat16().to(dev), torch.randn((E, n, k), generator=g).bfloat16().to(dev)
    w4, ws4 = packed(w4_raw(g, n, k, 32, True, E), 32, dev)
    od = offsets_of([rows // 2, 0, rows - rows // 2]).to(dev)
    run = lambda: (ops.ragged_mm(x, od, w), ops.ragged_mm_backward(x[:, :n].contiguous(), x, od, w)[0], ops.w4_mm(x, w4, ws4, n, k, 32, offsets=od))
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for counts, first in (([3, 1, 2], 1), ([0, rows, 0], 0), ([1, 0, 0], rows - 1), ([0, 0, 0], 0)):
        od.copy_(offsets_of(counts, first))
        graph.replay()
        torch.cuda.synchronize()
        rest = none_of(od.cpu(), rows)
        for o, want in zip(outs, run()):
            assert torch.equal(o, want) and not o[rest].any()
