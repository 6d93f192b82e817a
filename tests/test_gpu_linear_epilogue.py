"""GPU parity of linear with bias, activation and residual: with act "none" the output is bit for bit the f32 product (the call
without them) plus the bias, plus the residual, rounded once to y's type; with an activation it is within the f32 error of the
activation of those values. The products against 64 bits at every operand and format; those of the framework's other kernels
equal the plain call's bit for bit."""
import numpy as np
import pytest
import torch

from sublayer import ACTS, U8, U24, Weight, act64, act_tol, close, f64, mxfp8_values, q8_values, rows, vec

pytestmark = pytest.mark.gpu

# operand, format, tokens, n, k: every kernel family (matvecs one token and a group, K-sliced, tiled, int8 MFMA; GEMM tiles of
# each workgroup shape and the K-split dense kernel; scaled MFMA), ragged rows and columns
CASES = [("q8", "q4_k", 1, 520, 4096), ("q8", "q4_k", 3, 129, 768), ("q8", "q4_k", 9, 4100, 1280), ("q8", "q4_k", 20, 2056, 8192),
         ("q8", "q6_k", 1, 77, 2560), ("q8", "q6_k", 5, 1000, 768), ("q8", "q4_0", 2, 33, 64), ("q8", "q4_kt", 1, 512, 2048),
         ("q8", "q4_kt", 8, 48, 4096), ("q8", "q4_kt", 33, 1040, 1536), ("q8", "q4_0t", 4, 64, 1024), ("q8", "mxfp4s", 3, 65, 320),
         ("q8", "q4_k", 70, 64, 256), ("q8", "q4_k", 2, 64, 8192),
         ("bf16", "q4_k", 2, 77, 4096), ("bf16", "q4_k", 3, 65, 512), ("bf16", "q4_0", 5, 130, 640), ("f32", "q6_k", 2, 31, 512),
         ("f32", "q4_0t", 3, 64, 2048), ("bf16", "mxfp4", 4, 50, 2880), ("f32", "mxfp4s", 1, 50, 2880), ("f32", "q4_0", 5, 6144, 2048), ("f32", "q4_k", 17, 100, 768),
         ("bf16", "q6_k", 33, 515, 1280), ("f32", "mxfp4", 63, 40, 960), ("f32", "mxfp4s", 16, 129, 640), ("q8", "q6_k", 40, 4100, 512),
         ("q8", "q4_0", 63, 100, 192), ("q8", "mxfp4s", 17, 77, 64), ("bf16", "mxfp4", 2, 20, 96), ("bf16", "q6_k", 1, 30, 256),
         ("f16", "q4_k", 100, 300, 512), ("f16", "q4_k", 333, 4096, 1024), ("f16", "q4_k", 64, 130, 256), ("f16", "q4_k", 1, 77, 768),
         ("f16", "q4_kt", 130, 144, 1024), ("f16", "q6_k", 65, 1030, 768), ("f16", "q6_k", 513, 2100, 256), ("f16", "q4_0", 200, 257, 512),
         ("f16", "q6_k", 70, 96, 4096), ("mxfp8", "mxfp4s", 70, 129, 320), ("mxfp8", "mxfp4t", 3, 96, 2880), ("mxfp8", "mxfp4t", 130, 160, 256)]


def _operand(kind, rng, T, k, dev):
    """(x, keyword arguments of the call, values in 64 bits)."""
    import qmm.ops as ops
    x = rows(rng, (T, k), torch.float32, dev)
    if kind == "q8":
        xq = ops.quant_q8(x)
        return xq, {"tokens": T}, q8_values(xq, T, k)
    if kind == "f16":
        x16, s = ops.row_scale_f16(x * 1e5)   # an exponent that is not 0
        assert (s[:, 1] > 1).all()
        return x16, {"scales": s}, f64(x16) * f64(s[:, 1:])
    if kind == "mxfp8":
        c, s = ops.quant_mxfp8(x)
        return c, {"scales": s}, mxfp8_values(c, s)
    x = x.to({"f32": torch.float32, "bf16": torch.bfloat16}[kind])
    return x, {"q8": False}, f64(x)


def _product(kind, w, x, kw, T, n, k):
    """The plain call's f32 result."""
    import qmm.ops as ops
    if kind == "q8":
        return ops.mv_q8(w.fmt, w.w, x, n, k, tokens=T, ws=w.ws)
    if kind in ("bf16", "f32"):
        return ops.mv(w.fmt, w.w, x, n, k, ws=w.ws)
    return ops.gemm(w.fmt, "store", x, w.w, n, k, scales=kw["scales"], ws=w.ws)


@pytest.mark.parametrize("kind,fmt,T,n,k", CASES)
def test_epilogue(dev, kind, fmt, T, n, k):
    import qmm.ops as ops
    rng = np.random.default_rng(T + 3 * n + 7 * k)
    w = Weight(fmt, rng, n, k, dev)
    x, kw, xv = _operand(kind, rng, T, k, dev)
    y0 = ops.linear(fmt, x, w.w, n, k, ws=w.ws, out_dtype=torch.float32, **kw)
    # Q4_K in one round of workgroups: a kernel with four K-parts, the plain call's has two
    small = kind == "f16" and fmt in ("q4_k", "q4_kt") and -(-T // 64) * -(-n // (128 if k <= 2048 else 64)) <= 256
    if not small and (kind in ("f16", "mxfp8") or fmt in ("q4_kt", "q4_0t") or (T == 1 and (kind, fmt) != ("bf16", "q6_k")) or
                      (kind == "q8" and fmt == "q4_k")):
        assert torch.equal(y0, _product(kind, w, x, kw, T, n, k))
    # an f32 sum of k exact products: at most k additions, each off by at most half a step of sum |x w|
    W = torch.from_numpy(w.W16 if kind == "f16" else w.W)
    close(f64(y0), xv @ W.T, k * U24 * (xv.abs() @ W.abs().T), "product")
    bias = vec(rng, n, dev)
    span = float(y0.abs().max())
    for out in (torch.float32, torch.bfloat16):
        res = rows(rng, (T, n), torch.bfloat16 if out == torch.float32 else torch.float32, dev, span)
        for b, r in ((bias, res), (None, res), (bias, None), (None, None)):
            want = y0 if b is None else y0 + b
            want = (want if r is None else want + r.float()).to(out)
            got = ops.linear(fmt, x, w.w, n, k, ws=w.ws, bias=b, residual=r, out_dtype=out, **kw)
            assert got.dtype == out and torch.equal(got, want), (b is None, r is None, out)
    # the activations, on values spread over their bends by the bias (|product| of thousands for the scaled f16 rows)
    b = bias * 4
    pre = f64(y0 + b)
    for act in ACTS:
        a = act64(act, pre)
        tol = act_tol(act, pre, a)
        got = ops.linear(fmt, x, w.w, n, k, ws=w.ws, bias=b, act=act, out_dtype=torch.float32, **kw)
        close(f64(got), a, tol, act)
        res = rows(rng, (T, n), torch.bfloat16, dev)
        got = ops.linear(fmt, x, w.w, n, k, ws=w.ws, bias=b, act=act, residual=res, out_dtype=torch.bfloat16, **kw)
        want = a + f64(res)
        close(f64(got), want, tol + (U8 + U24) * (want.abs() + tol), act + " + residual")


def test_activations_over_their_range(dev):
    """Every activation at values from 1e-30 to the largest floats, infinities and NaN, through a product with one weight:
    x W^T = 0 (zero rows), so the bias is the argument."""
    import qmm.ops as ops
    mag = np.concatenate([10.0 ** np.arange(-30, 39, 1.0), np.linspace(0.01, 20, 400), [80, 88, 89, 100, 104, 3e38]])
    v = np.concatenate([-mag, mag, [0.0, -0.0, np.inf, -np.inf, np.nan]]).astype(np.float32)
    n = -(-v.size // 16) * 16
    b = torch.zeros(n)
    b[:v.size] = torch.from_numpy(v)
    w = Weight("q4_0", np.random.default_rng(3), n, 256, dev)
    x = torch.zeros((64, 256), dtype=torch.float16, device=dev)
    xr = torch.zeros((1, 256), device=dev)
    pre = b.double()
    fin = pre.isfinite()
    for act in ACTS:
        a = act64(act, pre)
        for got in (ops.linear("q4_0", x, w.w, n, 256, bias=b.to(dev), act=act)[:1],
                    ops.linear("q4_0", xr, w.w, n, 256, bias=b.to(dev), act=act, q8=False)):
            got = f64(got)[0]
            ok = fin & (a.abs() < 3.4e38)
            close(got[ok], a[ok], act_tol(act, pre, a)[ok], act)
            assert got[pre.isnan()].isnan().all(), act
            top = pre == float("inf")
            assert (got[top] == (1.0 if act == "sigmoid" else float("inf"))).all(), act


def test_residual_is_y_and_y_argument(dev):
    import qmm.ops as ops
    rng = np.random.default_rng(5)
    for kind, fmt, T, n, k in (("q8", "q4_k", 1, 264, 4096), ("q8", "q4_kt", 16, 4096, 1024), ("f16", "q4_k", 200, 260, 512),
                               ("f16", "q6_k", 200, 260, 512), ("mxfp8", "mxfp4t", 80, 96, 256), ("f32", "q6_k", 3, 96, 256)):
        w = Weight(fmt, rng, n, k, dev)
        x, kw, _ = _operand(kind, rng, T, k, dev)
        for dt in (torch.float32, torch.bfloat16):
            r = rows(rng, (T, n), dt, dev)
            want = ops.linear(fmt, x, w.w, n, k, ws=w.ws, residual=r, out_dtype=dt, act="silu", **kw)
            y = r.clone()
            got = ops.linear(fmt, x, w.w, n, k, ws=w.ws, residual=y, y=y, act="silu", **kw)
            assert got.data_ptr() == y.data_ptr() and torch.equal(got, want)


def test_rows_take_the_operands_path(dev):
    """f32 / bf16 rows: brought into the operand that linear multiplies, then the operand's call."""
    import qmm.ops as ops
    rng = np.random.default_rng(6)
    for fmt, T in (("q4_k", 1), ("q4_k", 63), ("q4_k", 64), ("q6_k", 65), ("q4_0", 4), ("q4_0", 90), ("q4_kt", 2), ("mxfp4s", 2),
                   ("mxfp4s", 64), ("mxfp4t", 3), ("q4_0t", 5), ("mxfp4", 3)):
        n, k = 96, 1024
        w = Weight(fmt, rng, n, k, dev)
        x, b = rows(rng, (T, k), torch.bfloat16, dev), vec(rng, n, dev)
        got = ops.linear(fmt, x, w.w, n, k, ws=w.ws, bias=b, out_dtype=torch.float32)
        if fmt == "mxfp4t":
            c, s = ops.quant_mxfp8(x)
            want = ops.gemm(fmt, "store", c, w.w, n, k, scales=s, ws=w.ws) + b
        else:
            want = ops.linear(fmt, x, w.w, n, k, ws=w.ws) + b
        # the same operand, so the same products; the sums of k = 1024 in another order differ by half steps of sum |x w|
        W = torch.from_numpy(w.W).abs()
        close(f64(got), f64(want), 2 * k * U24 * (f64(x).abs() * 1.01 @ W.T) + U24, fmt)


def test_padding_tiles_and_neighbour_rows(dev):
    """64-row tiles of padding rows keep their y; a row of NaN or infinities changes no other row; no bytes past y."""
    import qmm.ops as ops
    rng = np.random.default_rng(7)
    T, n, k = 200, 136, 512
    for fmt in ("q4_k", "q6_k"):
        w = Weight(fmt, rng, n, k, dev)
        x = rows(rng, (T, k), torch.bfloat16, dev)
        info = torch.ones((T, 4), dtype=torch.int32, device=dev)
        info[64:128] = 0
        x16, s = ops.row_scale_f16(x, info=info)
        b = vec(rng, n, dev)
        y = torch.full((T, n), 7.0, dtype=torch.bfloat16, device=dev)
        ops.linear(fmt, x16, w.w, n, k, scales=s, bias=b, y=y)
        full = ops.linear(fmt, *ops.row_scale_f16(x)[:1], w.w, n, k, scales=ops.row_scale_f16(x)[1], bias=b, out_dtype=torch.bfloat16)
        assert (y[64:128] == 7).all() and torch.equal(y[:64], full[:64]) and torch.equal(y[128:], full[128:])
        x2 = x.clone()
        x2[5] = float("nan")
        x2[150, 3] = float("inf")
        got = ops.linear(fmt, x2, w.w, n, k, bias=b, out_dtype=torch.bfloat16)
        keep = [i for i in range(T) if i not in (5, 150)]
        assert torch.equal(got[keep], full[keep]) and got[5].isnan().all()
        guard = torch.full((T * n + 64,), 3.0, device=dev)
        ops.linear(fmt, x, w.w, n, k, bias=b, y=guard[:T * n].view(T, n))
        assert (guard[T * n:] == 3).all()


@pytest.mark.parametrize("fmt,T,n,k", [("q4_k", 64, 136, 4096), ("q4_k", 333, 4096, 256), ("q4_k", 100, 300, 256), ("q4_kt", 130, 144, 1024),
                                       ("q6_k", 513, 2104, 256), ("q6_k", 70, 96, 4096), ("q4_0", 200, 264, 512), ("q6_k", 1500, 4104, 256),
                                       ("q4_k", 1300, 4104, 512)])
def test_rows_at_any_address(dev, fmt, T, n, k):
    """Rows of y, the residual and dy that do not start on 16 bytes take the same values as rows that do."""
    import qmm.ops as ops
    rng = np.random.default_rng(T + n)
    w, u, b = Weight(fmt, rng, n, k, dev), Weight(fmt, rng, n, k, dev), vec(rng, n, dev)
    x, s = ops.row_scale_f16(rows(rng, (T, k), torch.float32, dev))

    def at(off, t):
        buf = torch.full((T * n + 64,), 3.0, dtype=t.dtype, device=dev)
        buf[off:off + T * n] = t.reshape(-1)
        return buf, buf[off:off + T * n].view(T, n)

    for dt in (torch.float32, torch.bfloat16):
        res, dy = rows(rng, (T, n), dt, dev), rows(rng, (T, n), dt, dev, 1e-3)
        want = ops.linear(fmt, x, w.w, n, k, scales=s, bias=b, residual=res, act="silu", out_dtype=dt)
        gated = ops.ffn_gate_up(fmt, x, w.w, u.w, n, k, scales=s, bias=b, act="gelu", out_dtype=dt)
        grads = ops.ffn_gate_up_backward(fmt, x, w.w, u.w, dy, n, k, scales=s, bias=b)
        for off in (0, 1, 2, 8):
            buf, y = at(off, torch.zeros_like(res))
            ops.linear(fmt, x, w.w, n, k, scales=s, bias=b, residual=at(8 - off, res)[1], act="silu", y=y)
            assert torch.equal(y, want) and (buf[:off] == 3).all() and (buf[off + T * n:] == 3).all(), off
            buf, y = at(off, torch.zeros_like(res))
            ops.ffn_gate_up(fmt, x, w.w, u.w, n, k, scales=s, bias=b, act="gelu", y=y)
            assert torch.equal(y, gated) and (buf[:off] == 3).all() and (buf[off + T * n:] == 3).all(), off
            got = ops.ffn_gate_up_backward(fmt, x, w.w, u.w, at(off, dy)[1], n, k, scales=s, bias=b)
            assert all(torch.equal(p, q) for p, q in zip(got, grads)), off


@pytest.mark.parametrize("fmt", ["q4_k", "q6_k", "q4_0", "mxfp4", "mxfp4t"])
def test_bf16_y_of_the_prefill_products(dev, fmt):
    """A bf16 y without any of the epilogue's arguments is the GEMM's own output from 64 rows on, in every mode."""
    import qmm.ops as ops
    rng = np.random.default_rng(14)
    T, n, k = 70, 96, 512
    w, u, x = Weight(fmt, rng, n, k, dev), Weight(fmt, rng, n, k, dev), rows(rng, (T, k), torch.bfloat16, dev)
    gfmt, gw, gs, gu, gus = fmt, w.w, w.ws, u.w, u.ws
    if fmt == "mxfp4":
        gfmt, (gw, gs), (gu, gus) = "mxfp4s", ops.repack_mxfp4(w.w, n, k), ops.repack_mxfp4(u.w, n, k)
    for mode in ("store", "acc", "swiglu"):
        y = rows(rng, (T, n), torch.bfloat16, dev)
        z, two = y.clone(), mode == "swiglu"
        ops.linear(fmt, x, w.w, n, k, y=y, mode=mode, ws=w.ws, w2=u.w if two else None, ws2=u.ws if two else None)
        ops.gemm(gfmt, mode, x, gw, n, k, w2=gu if two else None, y=z, ws=gs, ws2=gus if two else None)
        assert torch.equal(y, z), mode
    got = ops.linear(fmt, x[:5], w.w, n, k, y=torch.empty((5, n), dtype=torch.bfloat16, device=dev), ws=w.ws)
    assert torch.equal(got, ops.linear(fmt, x[:5], w.w, n, k, ws=w.ws, out_dtype=torch.bfloat16))
