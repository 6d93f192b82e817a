"""GPU parity of linear_backward: dpre against the activation's slope in 64 bits at the argument's bounds, dx exactly the
transposed product of the dpre that came back, differences of the 64-bit forward, odd addresses, replays.

The argument is an f32 sum of k exact products, off by at most e = k half steps of sum |x w|; the slopes' own slopes are below
1.13, so dpre is off by 1.13 e |dy|, by a few hundred half steps of f32 of |dy| (the hardware's exponential and reciprocal),
and by its rounding to bf16."""
import numpy as np
import pytest
import torch

from sublayer import ACTS, U8, U24, Weight, act64, close, f64, rows, vec

pytestmark = pytest.mark.gpu

CASES = [("q4_k", 1, 64, 256), ("q4_k", 77, 768, 512), ("q4_k", 130, 333, 768), ("q4_k", 700, 4104, 512), ("q4_kt", 70, 144, 1024),
         ("q6_k", 65, 321, 512), ("q6_k", 3, 7, 256), ("q4_0", 77, 768, 256), ("q4_0", 129, 65, 768), ("q6_k", 1100, 2056, 256), ("q4_kt", 5, 16, 512)]


@pytest.mark.parametrize("fmt,T,n,k", CASES)
@pytest.mark.parametrize("act", ACTS)
def test_formula(dev, fmt, T, n, k, act):
    import qmm.ops as ops
    rng = np.random.default_rng(T + n + k)
    w, x = Weight(fmt, rng, n, k, dev), rows(rng, (T, k), torch.bfloat16, dev)
    dy = rows(rng, (T, n), torch.bfloat16 if T % 2 else torch.float32, dev, 1e-4)
    b = vec(rng, n, dev) if n % 2 == 0 else None
    dx, dpre = ops.linear_backward(fmt, x, w.w, dy, n, k, bias=b, act=act, out_dtype=torch.float32)
    assert torch.equal(dx, ops.gemm_t(fmt, dpre, w.w, n, k))
    if act == "none":
        assert dpre is dy
        return
    x16, s = ops.row_scale_f16(x)
    xv, W = f64(x16) * f64(s[:, 1:]), torch.from_numpy(w.W16)
    v = xv @ W.T + (f64(b) if b is not None else 0)
    e = k * U24 * (xv.abs() @ W.abs().T) + U24 * v.abs()
    z = v.clone().requires_grad_()
    (act64(act, z) * f64(dy)).sum().backward()
    tol = f64(dy).abs() * (1.13 * e + 200 * U24)
    tol = tol + U8 * (z.grad.abs() + tol) + 2.0 ** -126
    if act == "relu":   # on the kink both slopes are right
        tol = torch.where(v.abs() <= e, torch.full_like(tol, float("inf")), tol)
    assert dpre.dtype == torch.bfloat16
    close(f64(dpre), z.grad, tol, "dpre")
    dxb, again = ops.linear_backward(fmt, x16, w.w, dy, n, k, scales=s, bias=b, act=act)
    assert torch.equal(again, dpre) and torch.equal(dxb, dx.bfloat16())


@pytest.mark.parametrize("act", [a for a in ACTS if a != "relu"])
def test_differences(dev, act):
    """<dx, v> against the central difference of the 64-bit forward along v at the staged weights: the difference is off by about
    step^2 of the third derivative, dpre by its rounding to bf16 (2^-8 of each term)."""
    import qmm.ops as ops
    rng = np.random.default_rng(12)
    T, n, k, step = 5, 48, 256, 1e-4
    w, b, dy = Weight("q4_k", rng, n, k, dev), vec(rng, n, dev), rows(rng, (T, n), torch.float32, dev)
    W = torch.from_numpy(w.W16)
    x16, s = ops.row_scale_f16(rows(rng, (T, k), torch.float32, dev, 0.3 / float(W.norm(dim=1).mean())))
    dx, dpre = ops.linear_backward("q4_k", x16, w.w, dy, n, k, scales=s, bias=b, act=act, out_dtype=torch.float32)
    x, v = f64(x16) * f64(s[:, 1:]), torch.from_numpy(rng.standard_normal((T, k))) / float(W.norm(dim=1).mean())
    loss = lambda x: (f64(dy) * act64(act, x @ W.T + f64(b))).sum()   # noqa: E731
    want = (loss(x + step * v) - loss(x - step * v)) / (2 * step)
    bound = (f64(dpre) * (v @ W.T)).abs().sum()
    assert abs((f64(dx) * v).sum() - want) <= 2 * U8 * bound + 1e-6 * (f64(dy).abs() * (v @ W.T).abs()).sum()


def test_addresses_padding_and_replays(dev):
    import qmm.ops as ops
    rng = np.random.default_rng(13)
    T, n, k = 200, 264, 512
    for fmt in ("q4_k", "q6_k"):
        w, b, x = Weight(fmt, rng, n, k, dev), vec(rng, n, dev), rows(rng, (T, k), torch.bfloat16, dev)
        x16, s = ops.row_scale_f16(x)
        for dt in (torch.float32, torch.bfloat16):
            dy = rows(rng, (T, n), dt, dev, 1e-3)
            want = ops.linear_backward(fmt, x16, w.w, dy, n, k, scales=s, bias=b, act="gelu")
            for off in (1, 2, 8):
                buf = torch.empty(T * n + 16, dtype=dt, device=dev)
                buf[off:off + T * n] = dy.reshape(-1)
                got = ops.linear_backward(fmt, x16, w.w, buf[off:off + T * n].view(T, n), n, k, scales=s, bias=b, act="gelu")
                assert all(torch.equal(p, q) for p, q in zip(got, want))
        bad = x.clone()
        bad[9] = float("nan")
        got = ops.linear_backward(fmt, bad, w.w, dy, n, k, bias=b, act="gelu")
        keep = [i for i in range(T) if i != 9]
        assert torch.equal(got[0][keep], want[0][keep]) and got[1][9].isnan().all()
        graph, gx = torch.cuda.CUDAGraph(), x16.clone()
        with torch.cuda.graph(graph):
            out = ops.linear_backward(fmt, gx, w.w, dy, n, k, scales=s, bias=b, act="gelu")
        other = ops.row_scale_f16(rows(rng, (T, k), torch.bfloat16, dev))[0]
        for src in (other, x16, other):
            gx.copy_(src)
            graph.replay()
            assert all(torch.equal(p, q) for p, q in zip(out, ops.linear_backward(fmt, src, w.w, dy, n, k, scales=s, bias=b, act="gelu")))
