"""GPU parity of rms_norm_backward: the formula in 64 bits, differences of the 64-bit norm, odd shapes and types, the
update in place, and the backward chain of a feed-forward sub-layer against autograd in 64 bits.

With hn = h r, M = mean |weight dy hn|: r's relative error is half that of a sum of squares, at most the additions on a path
(n = 42 + k / 256, as for the forward norm) in half steps, and six more; the mean's terms and sum add n + 6 half steps of M;
each of the two parts takes r once more and three products. So |dx| is off by at most 2 (n + 8) half steps of
r |weight dy| + r |hn| M, and two additions of |dx| itself. A column's sum over the rows has at most rows / 512 + 16 + 64
additions on a path and terms with r's error."""
import numpy as np
import pytest
import torch

from helpers import assert_close_rel_l2
from sublayer import U8, U24, Weight, close, f64, rows, vec

pytestmark = pytest.mark.gpu
EPS = 1e-6
DT = {"f32": torch.float32, "bf16": torch.bfloat16, None: None}


def _want(h, w, dy, dh, eps=EPS):
    h, w, dy = f64(h), f64(w), f64(dy)
    r = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    hn, g = h * r, w * dy
    m = (g * hn).mean(-1, keepdim=True)
    dx = r * (g - hn * m) + (f64(dh) if dh is not None else 0)
    n = 42 + h.shape[1] / 256
    M = (g * hn).abs().mean(-1, keepdim=True)
    tol = 2 * (n + 8) * U24 * r * (g.abs() + hn.abs() * M) + 4 * U24 * dx.abs()
    return dx, tol, (dy * hn).sum(0), ((n / 2 + 12) + h.shape[0] / 512 + 80) * U24 * (dy * hn).abs().sum(0)


@pytest.mark.parametrize("T,k", [(1, 4096), (3, 128), (17, 8), (65, 1), (5, 7), (2, 2047), (9, 2880), (33, 512), (2, 520), (1100, 64),
                                 (4, 8192), (3, 12800), (1, 16392), (2, 32768), (1, 32767), (300, 256), (1500, 2880), (700, 333), (8300, 128)])
@pytest.mark.parametrize("x,dt,dh", [("bf16", "bf16", "bf16"), ("f32", "f32", None), ("f32", "bf16", "f32")])
def test_formula(dev, T, k, x, dt, dh):
    import qmm.ops as ops
    rng = np.random.default_rng(T + k)
    h, dy = rows(rng, (T, k), DT[x], dev, 2.0), rows(rng, (T, k), DT[dt], dev, 1e-3)
    dht = rows(rng, (T, k), DT[dh], dev, 1e-3) if dh else None
    w = (1 + vec(rng, k, dev, 0.2)).to(torch.bfloat16 if T % 2 else torch.float32)
    want, tol, dw, dw_tol = _want(h, w, dy, dht)
    got, gw = ops.rms_norm_backward(h, w, dy, EPS, dh=dht, out_dtype=torch.float32)
    close(f64(got), want, tol, "dx")
    close(f64(gw), dw, dw_tol, "dweight")
    gb, none = ops.rms_norm_backward(h, w, dy, EPS, dh=dht, out_dtype=torch.bfloat16, dweight=False)
    assert none is None and torch.equal(gb, got.bfloat16())
    if dht is not None:   # into dh's own rows
        rows_out, gw2 = ops.rms_norm_backward(h, w, dy, EPS, dh=dht, dx=dht)
        assert rows_out is dht and torch.equal(dht, got.to(dht.dtype)) and torch.equal(gw2, gw)


def test_differences(dev):
    """Central differences of sum(dy y) + sum(dh h) in 64 bits: their error is about step^2, 1e-8 of the gradients' size."""
    import qmm.ops as ops
    rng = np.random.default_rng(4)
    T, k, step = 3, 40, 1e-4
    x, w = rows(rng, (T, k), torch.float32, dev), 1 + vec(rng, k, dev, 0.3)
    dy, dh = rows(rng, (T, k), torch.float32, dev), rows(rng, (T, k), torch.float32, dev)
    dx, dw = ops.rms_norm_backward(x, w, dy, EPS, dh=dh)

    def loss(x, w):
        y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        return (f64(dy) * y).sum() + (f64(dh) * x).sum()

    for t in range(T):
        for c in range(0, k, 7):
            e = torch.zeros(T, k, dtype=torch.float64)
            e[t, c] = step
            d = (loss(f64(x) + e, f64(w)) - loss(f64(x) - e, f64(w))) / (2 * step)
            assert abs(d - f64(dx)[t, c]) < 1e-5
            d = (loss(f64(x), f64(w) + e[t]) - loss(f64(x), f64(w) - e[t])) / (2 * step)
            assert abs(d - f64(dw)[c]) < 1e-5


def test_rows_at_any_address_and_other_rows(dev):
    import qmm.ops as ops
    rng = np.random.default_rng(5)
    T, k = 40, 264
    h, dy, w = rows(rng, (T, k), torch.bfloat16, dev), rows(rng, (T, k), torch.bfloat16, dev), 1 + vec(rng, k, dev, 0.2)
    want, tol, dw, dw_tol = _want(h, w, dy, None)
    full, fw = ops.rms_norm_backward(h, w, dy, EPS, out_dtype=torch.float32)
    for off in (1, 2, 4):
        buf = torch.full((T * k + 16,), 3.0, device=dev)
        hb = torch.empty(T * k + 16, dtype=torch.bfloat16, device=dev)
        hb[off:off + T * k] = h.reshape(-1)
        got, gw = ops.rms_norm_backward(hb[off:off + T * k].view(T, k), w, dy, EPS, dx=buf[off:off + T * k].view(T, k))
        close(f64(got), want, tol, "dx")
        close(f64(gw), dw, dw_tol, "dweight")
        assert (buf[:off] == 3).all() and (buf[off + T * k:] == 3).all()
    bad = h.clone()
    bad[7] = float("nan")
    bad[20, 3] = float("inf")
    got, gw = ops.rms_norm_backward(bad, w, dy, EPS, out_dtype=torch.float32)
    keep = [i for i in range(T) if i not in (7, 20)]
    assert torch.equal(got[keep], full[keep]) and got[7].isnan().all() and gw.isnan().all()
    zero, zw = ops.rms_norm_backward(torch.zeros_like(h), w, dy, EPS, out_dtype=torch.float32)
    close(f64(zero), f64(w) * f64(dy) * 1e3, 16 * U24 * (f64(w) * f64(dy) * 1e3).abs(), "rows of zeros")   # 1 / sqrt(eps)
    assert (zw == 0).all()


def _backward(layer, x16, s, h, dh, act, T):
    import qmm.ops as ops
    gate, up, down, norm, H, F = layer
    da = ops.gemm_t(down.fmt, dh, down.w, H, F, out_dtype=torch.bfloat16)
    dn, dgu = ops.ffn_gate_up_backward(gate.fmt, x16, gate.w, up.w, da, F, H, scales=s, act=act)
    return ops.rms_norm_backward(h, norm, dn, EPS, dh=dh) + (dgu,)


@pytest.mark.parametrize("fmt,down,T,act", [("q4_k", "q6_k", 70, "silu"), ("q4_0", "q4_0", 5, "gelu"), ("q4_kt", "q4_kt", 130, "swiglu_oai")])
def test_backward_of_a_sublayer(dev, fmt, down, T, act):
    """Forward to the block's output rows and all the way back, against autograd in 64 bits; replayed from a graph. bf16 rows
    between the steps (da, dgu, dn: 2^-9 rms each over sqrt 3) and the f16 operands: rel-L2 below 1e-2 of the block's part."""
    import qmm.ops as ops
    rng = np.random.default_rng(T)
    H, F = 512, 1024
    gate, up, dn = Weight(fmt, rng, F, H, dev), Weight(fmt, rng, F, H, dev), Weight(down, rng, H, F, dev)
    norm = 1 + vec(rng, H, dev, 0.1)
    x, r, dh = (rows(rng, (T, H), torch.bfloat16, dev, v) for v in (1.0, 1.0, 1e-3))
    x16, s, h = ops.rms_norm(x, norm, EPS, residual=r, out="f16")
    a = ops.ffn_gate_up(fmt, x16, gate.w, up.w, F, H, act=act, scales=s, out_dtype=torch.bfloat16)
    ops.linear(down, a, dn.w, H, F, residual=h, out_dtype=torch.bfloat16)
    layer = (gate, up, dn, norm, H, F)
    dx, dw, dgu = _backward(layer, x16, s, h, dh, act, T)

    hd, nd = f64(h).requires_grad_(), f64(norm).requires_grad_()
    y = hd / torch.sqrt(hd.square().mean(-1, keepdim=True) + EPS) * nd
    # the projections of the f16 operand on the staged weights, as the kernels take them: a clamp's slope is 0 or 1, so with
    # arguments off by the operand's rounding (2^-11 of |u| of some tens) a part in 4000 would fall on a limit's other side,
    # which alone is sqrt(1 / 4000 / 0.2) = 3.5e-2 of the gradient where a fifth of the arguments lie inside
    y = y + (f64(x16) * f64(s[:, 1:]) - y).detach()
    W = lambda w: torch.from_numpy(w.W16)   # noqa: E731
    g, u = y @ W(gate).T, y @ W(up).T
    if act == "swiglu_oai":
        gc = g.clamp(max=7.0)
        a = gc * torch.sigmoid(1.702 * gc) * (u.clamp(-7.0, 7.0) + 1)
    elif act == "silu":
        a = g * torch.sigmoid(g) * u
    else:
        a = torch.nn.functional.gelu(g, approximate="tanh") * u
    (a @ W(dn).T).backward(f64(dh))   # the block's part; the residual's is dh itself
    assert_close_rel_l2(f64(dx).numpy() - f64(dh).numpy(), hd.grad.numpy(), 2e-2, "dx")
    assert_close_rel_l2(f64(dw).numpy(), nd.grad.numpy(), 2e-2, "dweight")

    graph = torch.cuda.CUDAGraph()
    gx, gh, gd = x16.clone(), h.clone(), dh.clone()
    with torch.cuda.graph(graph):
        out = _backward(layer, gx, s, gh, gd, act, T)
    for k in (1.0, 0.5, 1.0):
        gd.copy_(dh * k)
        graph.replay()
        want = _backward(layer, x16, s, h, dh * k, act, T)
        assert all(torch.equal(p, q) for p, q in zip(out, want))
