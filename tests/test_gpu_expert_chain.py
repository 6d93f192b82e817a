"""Expert layers of the 4-bit and ragged products as a user's program runs them: routed, sorted, multiplied, combined, and their
gradients, against the same layer in 64 bits; the products on other streams, at the limits of the experts' number, on rows that all
go to one expert; the integration document's example as it stands."""
import os
import re

import pytest
import torch

from qmm import ops
from ragged_case import U, Guarded, by_expert, gen, held, offsets_of, w4_raw
from test_gpu_w4 import packed

pytestmark = pytest.mark.gpu
DOC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")


def routed(ids, E):
    """(rows of the assignments sorted by expert, offsets) on the device, as the example sorts them."""
    order = torch.sort(ids.view(-1), stable=True)
    return order.indices, torch.searchsorted(order.values, torch.arange(E + 1, device=ids.device, dtype=ids.dtype)).int()


def rel(got, want):
    return float((got.cpu().double() - want).norm() / want.norm())


@pytest.mark.parametrize("T,E,KU", [(1, 8, 2), (13, 128, 8), (300, 16, 4)])
def test_four_bit_experts(dev, T, E, KU):
    """gate and up in one product, down in another, silu between. The up product's operand is f16 or exact, the activation is rounded
    to bf16 once (2^-8 / sqrt 3 of a value at most, rms) and the two products' weights and outputs to f16 and f32: rel-L2 below
    2^-8 / sqrt 3 + 4 2^-11 together, 4.3e-3."""
    H, F, g = 256, 160, gen(T)
    gu, dn = w4_raw(g, 2 * F, H, 64, True, E), w4_raw(g, H, F, 32, False, E)
    x, logits = torch.randn((T, H), generator=g).bfloat16(), torch.randn((T, E), generator=g)
    gu_w, dn_w = packed(gu, 64, dev), packed(dn, 32, dev)
    ids, wts = ops.moe_topk(logits.to(dev), KU, gating=1, norm=True)
    rows, offsets = routed(ids, E)
    a = ops.w4_mm(x.to(dev)[rows // KU], *gu_w, 2 * F, H, 64, offsets=offsets)
    a = (torch.nn.functional.silu(a[:, :F]) * a[:, F:]).bfloat16()
    y = ops.w4_mm(a, *dn_w, H, F, 32, offsets=offsets)
    out = torch.zeros((T, H), device=dev).index_add_(0, rows // KU, y * wts.view(-1)[rows][:, None])
    want, xd = torch.zeros((T, H), dtype=torch.float64), x.double()
    for t in range(T):
        for e, p in zip(ids[t].tolist(), wts[t].tolist()):
            u = gu[3][e] @ xd[t]
            want[t] += p * (dn[3][e] @ (torch.nn.functional.silu(u[:F]) * u[F:]))
    assert rel(out, want) < 4.3e-3


@pytest.mark.parametrize("T,E,KU", [(5, 4, 2), (200, 12, 3)])
def test_training_step_of_experts(dev, T, E, KU):
    """The layer's gradients with respect to x and both weights against autograd in 64 bits at the same bf16 values. Every product's
    output is rounded to bf16 once (at most 2^-8 of a value) and meets two more such roundings on the way back: rel-L2 below 3 2^-8."""
    H, F, g = 96, 136, gen(T)
    x, ids = torch.randn((T, H), generator=g).bfloat16(), torch.stack([torch.randperm(E, generator=g)[:KU] for _ in range(T)]).int()
    up, dn = (torch.randn((E, *s), generator=g).div(s[1] ** 0.5).bfloat16() for s in ((F, H), (H, F)))
    dy = torch.randn((T, H), generator=g).bfloat16()
    rows, offsets = routed(ids.to(dev), E)
    xs, upd, dnd = x.to(dev)[rows // KU], up.to(dev), dn.to(dev)
    h = ops.ragged_mm(xs, offsets, upd)
    a = torch.relu(h)
    y = torch.zeros((T, H), device=dev).index_add_(0, rows // KU, ops.ragged_mm(a, offsets, dnd, out_dtype=torch.float32))
    da, ddn = ops.ragged_mm_backward(dy.to(dev)[rows // KU], a, offsets, dnd, dw_dtype=torch.float32)
    dxs, dup = ops.ragged_mm_backward(da * (h > 0), xs, offsets, upd, dw_dtype=torch.float32)
    dx = torch.zeros((T, H), device=dev).index_add_(0, rows // KU, dxs.float())

    xd, upl, dnl = x.double().requires_grad_(), up.double().requires_grad_(), dn.double().requires_grad_()
    r, o = rows.cpu(), offsets.cpu().tolist()
    parts = []
    for e in range(E):
        he = xd[r[o[e]:o[e + 1]] // KU] @ upl[e].t()
        parts.append((he * (h[o[e]:o[e + 1]].cpu() > 0)) @ dnl[e].t())   # the kernel's own signs: a rounding may move one
    want = torch.zeros((T, H), dtype=torch.float64).index_add(0, r // KU, torch.cat(parts))
    want.backward(dy.double())
    for name, got, ref in (("y", y, want.detach()), ("dx", dx, xd.grad), ("up", dup, upl.grad), ("down", ddn, dnl.grad)):
        assert rel(got, ref) < 3 * 2.0 ** -8, name


def test_example(dev):
    """The document's block as it stands. Few rows and f32 results: only f32 sums and, for dw, the products' own order."""
    block = [b for b in re.findall(r"^```python\n(.*?)^```", open(DOC).read(), flags=re.S | re.M) if "ops.w4_pack(" in b]
    assert len(block) == 1
    T, E, KU, n, k, g = 9, 4, 2, 48, 256, gen(1)
    dense, experts = w4_raw(g, n, k, 128), w4_raw(g, n, k, 128, True, E)
    w_experts, ws_experts = packed(experts, 128, dev)
    x, w16 = torch.randn((T, k), generator=g).bfloat16(), torch.randn((E, n, k), generator=g).bfloat16()
    dys = torch.randn((T * KU, n), generator=g).bfloat16()
    ids = torch.stack([torch.randperm(E, generator=g)[:KU] for _ in range(T)]).int()
    names = dict(ops=ops, torch=torch, codes=dense[0].to(dev), scales=dense[1].to(dev), zeros=dense[2].to(dev), x=x.to(dev), n=n, k=k, E=E,
                 KU=KU, ids=ids.to(dev), w_experts=w_experts, ws_experts=ws_experts, w16=w16.to(dev), dys=dys.to(dev))
    exec(block[0], names)
    held(names["y"], x.double() @ dense[3].t(), (k + 8) * U * (x.double().abs() @ dense[4].t()))
    offsets, xs = names["offsets"].cpu(), names["xs"].cpu().double()
    assert offsets.tolist() == [int((ids < e).sum()) for e in range(E + 1)]
    held(names["ys"], by_expert(xs, w16.double(), offsets), k * U * by_expert(xs.abs(), w16.double().abs(), offsets))
    held(names["dxs"], by_expert(dys.double(), w16.double(), offsets, t=True), n * U * by_expert(dys.double().abs(), w16.double().abs(), offsets, t=True))
    o = offsets.tolist()
    want = torch.stack([dys[a:b].double().t() @ xs[a:b] for a, b in zip(o, o[1:])])
    held(names["dw"], want, T * KU * U * torch.stack([dys[a:b].double().abs().t() @ xs[a:b].abs() for a, b in zip(o, o[1:])]))


def test_calls_on_two_streams(dev):
    """Calls that overlap, sums in parts and in one: each has its own workspace."""
    g = gen(7)
    raw = w4_raw(g, 72, 8192, 128)
    w, ws = packed(raw, 128, dev)
    x = [torch.randn((90, 8192), generator=g).bfloat16().to(dev) for _ in range(2)]
    r, rw = torch.randn((7000, 64), generator=g).bfloat16().to(dev), torch.randn((7000, 72), generator=g).bfloat16().to(dev)
    offsets = offsets_of([7000]).to(dev)
    run = lambda i: (ops.w4_mm(x[i], w, ws, 72, 8192, 128), ops.ragged_mm_dw(rw, r, offsets, out_dtype=torch.float32))
    want = [run(0), run(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(o, want[i]))


def test_two_graphs(dev):
    """Two captured calls whose sums are taken in parts, replayed in turn and again after eager work."""
    g = gen(8)
    raw = w4_raw(g, 64, 8192, 64)
    w, ws = packed(raw, 64, dev)
    x = [torch.randn((80, 8192), generator=g).bfloat16().to(dev) for _ in range(2)]
    want = [ops.w4_mm(v, w, ws, 64, 8192, 64) for v in x]
    graphs, outs = [], []
    for v in x:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.w4_mm(v, w, ws, 64, 8192, 64))
        graphs.append(graph)
    for _ in range(3):
        for o in outs:
            o.zero_()
        for graph in graphs:
            graph.replay()
        assert torch.equal(ops.w4_mm(x[0], w, ws, 64, 8192, 64), want[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_most_experts(dev):
    """1024 experts, most of them empty: 16 a lane of the search for a tile's expert."""
    g, E, n, k = gen(3), 1024, 16, 32
    counts = [int(c) for c in torch.randint(0, 3, (E,), generator=g)]
    counts[777], counts[1023] = 300, 70
    rows, offsets = sum(counts) + 4, offsets_of(counts, 1)
    x, dy = torch.randn((rows, k), generator=g).bfloat16(), torch.randn((rows, n), generator=g).bfloat16()
    raw, w16 = w4_raw(g, n, k, 32, True, E), torch.randn((E, n, k), generator=g).bfloat16()
    w, ws = packed(raw, 32, dev)
    live = slice(1, rows - 3)
    x[0], x[rows - 3:], dy[0], dy[rows - 3:] = (float("nan"),) * 4
    y, y16, yr, dx, dxr = (Guarded((rows, c), torch.float32, dev) for c in (n, n, n, k, k))
    xd, od = x.to(dev), offsets.to(dev)
    ops.w4_mm(xd, w, ws, n, k, 32, offsets=od, y=y.t)                       # few rows an expert
    x16, scales = ops.row_scale_f16(xd.nan_to_num())
    ops.w4_mm(x16, w, ws, n, k, 32, offsets=od, scales=scales, y=y16.t)
    ops.ragged_mm(xd, od, w16.to(dev), y=yr.t)
    ops.w4_mm_t(dy.nan_to_num().to(dev), w, ws, n, k, 32, offsets=od, y=dx.t)
    ops.ragged_mm_t(dy.to(dev), od, w16.to(dev), dx=dxr.t)
    dw = ops.ragged_mm_dw(dy.to(dev), xd, od, out_dtype=torch.float32)
    for v in (y, y16, yr, dx, dxr):
        v.check(kept=((0, 1), (rows - 3, rows)))
    xa, da = x.double(), dy.double()
    want, size = by_expert(xa, raw[3], offsets)[live], by_expert(xa.abs(), raw[4], offsets)[live]
    held(y.t[live], want, (k + 8) * U * size)
    held(y16.t[live], want, (2.0 ** -11 + k * U) * size + 1e-9)   # 2^-38 max |row| sum |w| is below 1e-9 here
    held(yr.t[live], by_expert(xa, w16.double(), offsets)[live], k * U * by_expert(xa.abs(), w16.double().abs(), offsets)[live])
    size = by_expert(da.abs(), raw[3].abs(), offsets, t=True)[live]
    held(dx.t[live], by_expert(da, raw[3], offsets, t=True)[live], (2.0 ** -11 + n * U) * size + 1e-9)
    held(dxr.t[live], by_expert(da, w16.double(), offsets, t=True)[live], n * U * by_expert(da.abs(), w16.double().abs(), offsets, t=True)[live])
    o = offsets.tolist()
    held(dw, torch.stack([da[a:b].t() @ xa[a:b] for a, b in zip(o, o[1:])]),
         300 * U * torch.stack([da[a:b].abs().t() @ xa[a:b].abs() for a, b in zip(o, o[1:])]))


@pytest.mark.parametrize("rows,E,n,k", [(60, 40, 72, 160), (500, 3, 16, 64), (250, 200, 24, 96), (31, 8, 400, 32)])
def test_every_row_one_experts(dev, rows, E, n, k):
    """A segment of all rows among empty ones: the few-row kernels walk it in layers of the grid, or one after the other."""
    g = gen(rows)
    offsets = torch.tensor([0] * (E // 2 + 1) + [rows] * (E - E // 2), dtype=torch.int32)
    raw, w16 = w4_raw(g, n, k, 32, True, E), torch.randn((E, n, k), generator=g).bfloat16()
    w, ws = packed(raw, 32, dev)
    x = torch.randn((rows, k), generator=g).bfloat16()
    for out in (torch.float32, torch.bfloat16):
        y, yr = Guarded((rows, n), out, dev), Guarded((rows, n), out, dev)
        ops.w4_mm(x.to(dev), w, ws, n, k, 32, offsets=offsets.to(dev), y=y.t)
        ops.ragged_mm(x.to(dev), offsets.to(dev), w16.to(dev), y=yr.t)
        y.check(), yr.check()
        size = by_expert(x.double().abs(), raw[4], offsets)
        held(y.t, by_expert(x.double(), raw[3], offsets), (2.0 ** -11 + (k + 8) * U) * size + 1e-8)   # 2^-38 max |row| sum |w| is below 1e-8
        held(yr.t, by_expert(x.double(), w16.double(), offsets), k * U * by_expert(x.double().abs(), w16.double().abs(), offsets))


def test_an_expert_does_not_see_its_neighbours(dev):
    """NaN and infinities of one expert's rows stay in its outputs and its weights' gradient."""
    g, n, k, E = gen(6), 72, 128, 3
    offsets = offsets_of([70, 65, 90])
    x, dy, w16 = (torch.randn(s, generator=g).bfloat16().to(dev) for s in ((225, k), (225, n), (E, n, k)))
    raw = w4_raw(g, n, k, 32, True, E)
    w, ws = packed(raw, 32, dev)
    od = offsets.to(dev)
    run = lambda: (ops.ragged_mm(x, od, w16), ops.ragged_mm_t(dy, od, w16), ops.w4_mm(x, w, ws, n, k, 32, offsets=od), ops.w4_mm_t(dy, w, ws, n, k, 32, offsets=od))
    clean, dw = run(), ops.ragged_mm_dw(dy, x, od)
    x[70:135], dy[70:135, ::2], dy[70:135, 1::2] = float("nan"), float("inf"), float("nan")
    for got, want in zip(run(), clean):
        assert torch.equal(got[:70], want[:70]) and torch.equal(got[135:], want[135:]) and not got[70:135].isfinite().any()
    got = ops.ragged_mm_dw(dy, x, od)
    assert torch.equal(got[0], dw[0]) and torch.equal(got[2], dw[2]) and got[1].isnan().all()


def test_outputs_at_odd_addresses(dev):
    """y that starts at an element's multiple, not at sixteen bytes: the tiles' narrow stores."""
    g, n, k = gen(5), 64, 96
    raw = w4_raw(g, n, k, 32)
    w, ws = packed(raw, 32, dev)
    for rows, x_type in ((5, torch.float32), (130, torch.bfloat16)):
        x = torch.randn((rows, k), generator=g).to(x_type).to(dev)
        xa = x if rows < 64 else ops.row_scale_f16(x)[0]
        scales = None if rows < 64 else ops.row_scale_f16(x)[1]
        want = ops.w4_mm(xa, w, ws, n, k, 32, scales=scales)
        y = torch.full((rows * n + 2,), 3.0, device=dev)
        ops.w4_mm(xa, w, ws, n, k, 32, scales=scales, y=y[1:-1].view(rows, n))
        assert torch.equal(y[1:-1].view(rows, n), want) and y[0] == 3 and y[-1] == 3
    dy = torch.randn((33, n), generator=g).to(dev)
    dx = torch.full((33 * k + 2,), 3.0, device=dev)
    ops.w4_mm_t(dy, w, ws, n, k, 32, y=dx[1:-1].view(33, k))
    assert torch.equal(dx[1:-1].view(33, k), ops.w4_mm_t(dy, w, ws, n, k, 32)) and dx[0] == 3 and dx[-1] == 3


@pytest.mark.parametrize("parts,n", [(1, 78), (1, 257), (2, 127), (1, 2047), (2, 1023), (2, 1025), (1, 5012), (2, 4095), (1, 8191), (1, 8193)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_operand_of_odd_rows(dev, parts, n, dtype):
    """Rows that are no multiple of eight values long, at the lengths where they change kernels."""
    from qmm import _lib
    T, N = 5, -(-n // 64) * 64
    x = (torch.randn((T, parts, n), generator=gen(n)) * 1e-3).to(dtype).to(dev)
    x[1, parts - 1, n - 1] = 5.0
    x[2, 0, 0] = float("nan")
    x[3] = 0
    buf = torch.full((T * parts * N + 64,), 9.0, dtype=torch.float16, device=dev)
    x16, s = buf[:-64].view(T, parts, N), torch.empty((T, 2), device=dev)
    _lib.call("qmm_grad_operand", T, parts, n, x.data_ptr(), ops._dt(x), x16.data_ptr(), s.data_ptr(), ops._stream())
    rest = [0, 1, 3, 4]
    assert (x16[..., n:] == 0).all() and (buf[-64:] == 9).all()
    assert torch.equal(x16[rest][..., :n], (x.float() * s[:, :1, None]).half()[rest])
    assert x16[2, 0, 0].isnan() and x16[2, :, :n].isnan().sum() == 1 and s[1].tolist() == [2.0 ** 11, 2.0 ** -11]
    m = x.float().abs().amax((1, 2))[[0, 4]] * s[[0, 4], 0]
    assert ((m >= 2.0 ** 13) & (m < 2.0 ** 14)).all() and s[3, 0] == 1


# larger tiles, deep and not, whole sums and sums in parts (a case of every tile and type: tile_cases.py)
@pytest.mark.parametrize("counts,N,K", [([9000, 1, 0, 8300], 520, 40), ([4000, 0, 4500, 1, 8800], 264, 416), ([4142], 160, 6304),
                                        ([5000, 7001, 600], 32, 4352), ([4000, 0, 42], 136, 6624), ([11000, 0, 8801], 528, 40),
                                        ([30, 0, 45, 0, 0], 6648, 40), ([4182], 32, 2016), ([75, 0, 4], 40, 1160), ([9001, 0, 7600], 32, 40),
                                        ([2054], 32, 2120), ([131, 0, 250], 2048, 1000)])
@pytest.mark.parametrize("back", [False, True])
def test_larger_tiles(dev, counts, N, K, back):
    """N outputs a row, K values in their sums, forward and backward."""
    g, rows, E = gen(N + K), sum(counts) + 5, len(counts)
    offsets = offsets_of(counts, 2)
    x, w = torch.randn((rows, K), generator=g).bfloat16().to(dev), torch.randn((E, K, N) if back else (E, N, K), generator=g).bfloat16().to(dev)
    x[:2], x[-3:] = float("nan"), float("nan")
    y = Guarded((rows, N), torch.float32, dev)
    (ops.ragged_mm_t(x, offsets.to(dev), w, dx=y.t) if back else ops.ragged_mm(x, offsets.to(dev), w, y=y.t))
    y.check(kept=((0, 2), (rows - 3, rows)))
    want, size = by_expert(x.double(), w.double(), offsets.to(dev), t=back)[2:-3], by_expert(x.double().abs(), w.double().abs(), offsets.to(dev), t=back)[2:-3]
    held(y.t[2:-3], want, K * U * size, "tiles")


@pytest.mark.parametrize("counts,n,k", [([1700], 33, 7232), ([9000, 0, 10700], 40, 544), ([1570], 328, 4960), ([16418], 4340, 32),
                                        ([12000, 814], 2708, 32), ([16429], 36, 320)])
def test_larger_tiles_of_the_transposed_product(dev, counts, n, k):
    g, rows, E = gen(n + k), sum(counts) + 1, len(counts)
    offsets = offsets_of(counts, 1)
    raw = w4_raw(g, n, k, 64, True, E)
    w, ws = packed(raw, 64, dev)
    dy = torch.randn((rows, n), generator=g).bfloat16().to(dev)
    y = Guarded((rows, k), torch.float32, dev)
    ops.w4_mm_t(dy, w, ws, n, k, 64, offsets=offsets.to(dev), y=y.t)
    y.check(kept=((0, 1),))
    wd = raw[3].to(dev)
    want, size = by_expert(dy.double(), wd, offsets.to(dev), t=True)[1:], by_expert(dy.double().abs(), wd.abs(), offsets.to(dev), t=True)[1:]
    lost = 2.0 ** -38 * dy.double().abs().amax(-1, keepdim=True)[1:].cpu() * by_expert(torch.ones_like(dy, dtype=torch.float64), wd.abs(), offsets.to(dev), t=True)[1:]
    held(y.t[1:], want, (2.0 ** -11 + n * U) * size + lost, "transposed tiles")


@pytest.mark.parametrize("counts,n,k", [([10, 0, 14, 5, 1], 520, 3992), ([8750], 144, 2192), ([9000, 0, 7000, 1, 103], 136, 1208),
                                        ([5000, 796], 16, 2072), ([30], 2952, 1304), ([968], 16, 16), ([70, 1300], 72, 264)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_larger_tiles_of_the_weight_gradient(dev, counts, n, k, dtype):
    g, rows, E = gen(n + k), sum(counts) + 5, len(counts)
    offsets = offsets_of(counts, 2)
    x, dy = torch.randn((rows, k), generator=g).to(dtype).to(dev), (0.1 * torch.randn((rows, n), generator=g)).to(dtype).to(dev)
    x[:2], x[-3:], dy[:2], dy[-3:] = (float("nan"),) * 4
    dw = Guarded((E, n, k), torch.float32, dev)
    ops.ragged_mm_dw(dy, x, offsets.to(dev), dw=dw.t)
    dw.check()
    at = offsets.tolist()
    for e, (a, b) in enumerate(zip(at, at[1:])):
        xd, dd = x[a:b].double(), dy[a:b].double().t().contiguous()
        held(dw.t[e], torch.mm(dd, xd).cpu(), (b - a + 16) * U * torch.mm(dd.abs(), xd.abs()).cpu(), f"expert {e}")


@pytest.mark.parametrize("rows,n,k", [(130, 264, 96), (130, 261, 96), (5, 40, 64), (90, 67, 8192)])   # the last: a sum in parts
@pytest.mark.parametrize("shift", [1, 3, 7])
def test_bf16_outputs_at_any_address(dev, rows, n, k, shift):
    raw = w4_raw(gen(n), n, k, 32)
    w, ws = packed(raw, 32, dev)
    x = torch.randn((rows, k), generator=gen(rows)).bfloat16().to(dev)
    x16, scales = ops.row_scale_f16(x) if rows > 64 else (x, None)
    want = ops.w4_mm(x16, w, ws, n, k, 32, scales=scales, out_dtype=torch.bfloat16)
    buf = torch.full((rows * n + 16,), 3.0, dtype=torch.bfloat16, device=dev)
    y = buf[shift:shift + rows * n].view(rows, n)
    ops.w4_mm(x16, w, ws, n, k, 32, scales=scales, y=y)
    assert torch.equal(y, want) and (buf[:shift] == 3).all() and (buf[shift + rows * n:] == 3).all()


@pytest.mark.parametrize("counts,first,tail,n,k,group,x_type,out", [
    ([31], 0, 0, 150, 12128, 64, "f32", "bf16"), ([63], 0, 0, 64, 4096, 32, "f32", "f32"), ([32], 0, 0, 33, 12288, 128, "bf16", "f32"),
    ([5], 0, 0, 17, 12288, 1 << 20, "f32", "f32"), ([20, 0, 11], 2, 3, 40, 12288, 128, "f32", "f32"), ([31, 30], 0, 1, 24, 8192, 64, "f32", "bf16")])
def test_few_rows_in_parts(dev, counts, first, tail, n, k, group, x_type, out):
    from qmm import _lib
    T = {"f32": torch.float32, "bf16": torch.bfloat16}
    rows, E, g = first + sum(counts) + tail, len(counts), gen(n + k)
    assert _lib.load().qmm_w4_mm_workspace_size(rows, k, n, E, ops._DT[T[x_type]]) >= 2 * rows * n * 4
    offsets = offsets_of(counts, first)
    raw = w4_raw(g, n, k, group, True, E)
    w, ws = packed(raw, group, dev)
    x = torch.randn((rows, k), generator=g).to(T[x_type])
    x[:first], x[rows - tail:] = float("nan"), float("nan")
    for _ in range(2):
        y = Guarded((rows, n), T[out], dev)
        ops.w4_mm(x.to(dev), w, ws, n, k, group, offsets=offsets.to(dev), y=y.t)
        y.check(kept=((0, first), (rows - tail, rows)))
        live = slice(first, rows - tail)
        held(y.t[live], by_expert(x.double(), raw[3], offsets)[live], (k + 8) * U * by_expert(x.double().abs(), raw[4], offsets)[live], "few rows in parts")


# 64 x 256, 128 x 128 and 128 x 256 tiles, one turn of K and several with an odd end
@pytest.mark.parametrize("counts,n,k", [([11761], 781, 32), ([16389], 523, 32), ([19801], 519, 32), ([9000, 7, 7402], 551, 32),
                                        ([9000, 0, 7803], 645, 32), ([12655], 389, 416), ([19008], 259, 416), ([1540], 7828, 416)])
def test_larger_tiles_of_the_four_bit_product(dev, counts, n, k):
    g, rows, E = gen(n + k), sum(counts) + 5, len(counts)
    offsets = offsets_of(counts, 2)
    raw = w4_raw(g, n, k, 64, True, E)
    w, ws = packed(raw, 64, dev)
    x = torch.randn((rows, k), generator=g).bfloat16().to(dev)
    x16, scales = ops.row_scale_f16(x)
    x16[:2], x16[-3:] = float("nan"), float("inf")
    y = Guarded((rows, n), torch.float32, dev)
    ops.w4_mm(x16, w, ws, n, k, 64, offsets=offsets.to(dev), scales=scales, y=y.t)
    y.check(kept=((0, 2), (rows - 3, rows)))
    wd, xd, od = raw[3].to(dev), x16.double() * scales.double()[:, 1:], offsets.to(dev)
    held(y.t[2:-3], by_expert(xd, wd, od)[2:-3], ((2.0 ** -11 + k * U) * by_expert(xd.abs(), wd.abs(), od))[2:-3], "4-bit tiles")


# two and three row blocks a wave, the last workgroup with fewer, one to four tiles of tokens
@pytest.mark.parametrize("rows,n,k,group", [(2, 4200, 160, 32), (9, 4121, 288, 64), (20, 4200, 416, 1 << 20), (40, 4137, 160, 64), (5, 8300, 160, 128),
                                            (16, 8211, 288, 32), (31, 8300, 96, 64), (63, 8227, 160, 32)])
@pytest.mark.parametrize("x_type", ["bf16", "f32"])
def test_few_rows_of_many_columns(dev, rows, n, k, group, x_type):
    g, t = gen(rows + n), {"bf16": torch.bfloat16, "f32": torch.float32}[x_type]
    raw = w4_raw(g, n, k, group)
    w, ws = packed(raw, group, dev)
    x = torch.randn((rows, k), generator=g).to(t)
    y = Guarded((rows, n), torch.float32, dev)
    ops.w4_mm(x.to(dev), w, ws, n, k, group, y=y.t)
    y.check()
    held(y.t, x.double() @ raw[3].t(), (k + 8) * U * (x.double().abs() @ raw[4].t()), "few rows, many columns")


@pytest.mark.parametrize("E,most,n,k,group", [(256, 1, 170, 160, 32), (256, 1, 170, 288, 128), (40, 3, 136, 160, 64), (100, 4, 150, 96, 32), (60, 40, 200, 128, 64),
                                              (90, 90, 130, 160, 1 << 20)])
@pytest.mark.parametrize("x_type", ["bf16", "f32"])
def test_few_rows_of_many_experts(dev, E, most, n, k, group, x_type):
    g, t = gen(E + n), {"bf16": torch.bfloat16, "f32": torch.float32}[x_type]
    counts = [int(c) for c in torch.randint(0, most + 1, (E,), generator=g)]
    if most == 1:
        counts = [1 if i % 8 else 0 for i in range(E)]
        counts[3], counts[9] = 0, 2
    rows, offsets = sum(counts) + 3, offsets_of(counts, 1)
    raw = w4_raw(g, n, k, group, True, E)
    w, ws = packed(raw, group, dev)
    x = torch.randn((rows, k), generator=g).to(t)
    x[0], x[rows - 2:] = float("inf"), float("nan")
    y = Guarded((rows, n), torch.float32, dev)
    from qmm import _lib
    od, xd = offsets.to(dev), x.to(dev)
    need = _lib.load().qmm_w4_mm_workspace_size(rows, k, n, E, ops._DT[t])
    work = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    _lib.call("qmm_w4_mm", rows, k, n, group, E, od.data_ptr(), xd.data_ptr(), ops._DT[t], None, w.data_ptr(), ws.data_ptr(), y.t.data_ptr(),
              ops._DT[torch.float32], work.data_ptr(), need, ops._stream())   # few rows, whatever the number that the Python call would take
    y.check(kept=((0, 1), (rows - 2, rows)))
    live = slice(1, rows - 2)
    held(y.t[live], by_expert(x.double(), raw[3], offsets)[live], (k + 8) * U * by_expert(x.double().abs(), raw[4], offsets)[live], "few rows, many experts")
