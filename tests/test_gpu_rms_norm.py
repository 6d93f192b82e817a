"""GPU parity of rms_norm: y against 64 bits elementwise, the residual sum exactly, and every operand form bit for bit what
its quantizer gives for the f32 y.

Tolerance of the f32 y: the squares are positive, so the sum's relative error is at most the additions on a path (a lane's
chain of at most 32 values and 10 exchanges and LDS additions, or k / 256 + 12 in the kernel for any k) in half steps; the
square root halves it; the division, the root, its reciprocal, the two products and h's own addition add six."""
import numpy as np
import pytest
import torch

from sublayer import U8, U24, close, f64, rows, vec

pytestmark = pytest.mark.gpu
EPS = 1e-6
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _inputs(dev, T, k, x, res, weight="f32", seed=0):
    rng = np.random.default_rng(1000 * T + k + seed)
    xt = rows(rng, (T, k), DT[x], dev)
    rt = rows(rng, (T, k), DT[res], dev, 2.0) if res else None
    w = (1 + vec(rng, k, dev, 0.2)).to(DT[weight])
    return xt, rt, w


def _want(xt, rt, w, eps=EPS):
    h = f64(xt) + (f64(rt) if rt is not None else 0)
    return h, h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * f64(w)


@pytest.mark.parametrize("T,k", [(1, 4096), (3, 128), (17, 8), (65, 1), (5, 7), (2, 2047), (9, 2880), (33, 512), (2, 520),
                                 (4, 8192), (3, 12800), (1, 16392), (2, 32768), (1, 32767), (300, 256)])
@pytest.mark.parametrize("x,res", [("bf16", "bf16"), ("f32", None), ("f32", "bf16"), ("bf16", "f32")])
def test_rows(dev, T, k, x, res):
    import qmm.ops as ops
    xt, rt, w = _inputs(dev, T, k, x, res, weight="bf16" if T % 2 else "f32")
    h, want = _want(xt, rt, w)
    y, scales, ht = ops.rms_norm(xt, w, EPS, residual=rt, out="f32")
    assert scales is None and y.dtype == torch.float32
    close(f64(y), want, ((42 + k / 256) / 2 + 8) * U24 * want.abs(), "y")
    if rt is None:
        assert ht is None
    else:   # one f32 addition, one rounding to the residual's type
        h32 = xt.float() + rt.float()
        assert torch.equal(ht, h32.to(ht.dtype)) and ht.dtype == rt.dtype
    yb = ops.rms_norm(xt, w, EPS, residual=rt, out="bf16")[0]
    assert torch.equal(yb, y.bfloat16())
    x16, s = ops.rms_norm(xt, w, EPS, residual=rt, out="f16")[:2]
    x16w, sw = ops.row_scale_f16(y)
    assert torch.equal(x16.view(torch.int16), x16w.view(torch.int16)) and torch.equal(s, sw)


@pytest.mark.parametrize("T,k", [(1, 4096), (5, 32), (7, 96), (33, 2880), (2, 512), (3, 544), (2, 12288), (2, 32768)])
@pytest.mark.parametrize("x,res", [("bf16", "bf16"), ("f32", None)])
def test_eight_bit_operands(dev, T, k, x, res):
    import qmm.ops as ops
    xt, rt, w = _inputs(dev, T, k, x, res)
    y = ops.rms_norm(xt, w, EPS, residual=rt, out="f32")[0]
    assert torch.equal(ops.rms_norm(xt, w, EPS, residual=rt, out="q8")[0], ops.quant_q8(y))
    codes, scales, _ = ops.rms_norm(xt, w, EPS, residual=rt, out="mxfp8")
    cw, sw = ops.quant_mxfp8(y)
    assert torch.equal(codes, cw) and torch.equal(scales, sw)


def test_large_rows_scale_into_f16(dev):
    """Rows whose y passes f16's range take an exponent; rows of tiny values keep theirs."""
    import qmm.ops as ops
    xt, _, w = _inputs(dev, 4, 512, "f32", None)
    w = w * torch.tensor([1e6], device=dev)
    y = ops.rms_norm(xt, w, EPS, out="f32")[0]
    x16, s, _ = ops.rms_norm(xt, w, EPS, out="f16")
    x16w, sw = ops.row_scale_f16(y)
    assert torch.equal(x16.view(torch.int16), x16w.view(torch.int16)) and torch.equal(s, sw) and (s[:, 0] < 1).all()
    close(f64(x16) * f64(s[:, 1:]), f64(y), 2.0 ** -11 * f64(y).abs() + 2.0 ** -24 * f64(s[:, 1:]), "x16")


def test_in_place_and_misaligned(dev):
    """h into the residual and into x; rows that start at odd addresses take the kernel for any k."""
    import qmm.ops as ops
    for k in (2880, 2881):
        xt, rt, w = _inputs(dev, 6, k, "bf16", "bf16")
        y, _, h = ops.rms_norm(xt, w, EPS, residual=rt, out="bf16")
        for name in ("residual", "x"):
            x2, r2 = xt.clone(), rt.clone()
            y2, _, h2 = ops.rms_norm(x2, w, EPS, residual=r2, out="bf16", h=r2 if name == "residual" else x2)
            assert torch.equal(y2, y) and torch.equal(h2, h) and h2.data_ptr() == (r2 if name == "residual" else x2).data_ptr()
            assert torch.equal(x2 if name == "residual" else r2, xt if name == "residual" else rt)
    flat = torch.zeros(6 * 2880 + 1, dtype=torch.bfloat16, device=dev)
    xm = flat[1:].view(6, 2880)
    xt, _, w = _inputs(dev, 6, 2880, "bf16", None)
    xm.copy_(xt)
    got, want = ops.rms_norm(xm, w, EPS, out="f32")[0], _want(xt, None, w)[1]
    close(f64(got), want, ((42 + 2880 / 256) / 2 + 8) * U24 * want.abs(), "misaligned")
    with pytest.raises(Exception, match="misaligned"):
        ops.rms_norm(xm, w, EPS, out="q8")


def test_zero_rows_eps_and_other_rows_values(dev):
    """A row of zeros is zeros; an infinity or NaN stays in its row."""
    import qmm.ops as ops
    xt, rt, w = _inputs(dev, 9, 2048, "f32", "f32")
    clean = ops.rms_norm(xt, w, EPS, residual=rt, out="f32")[0]
    xt[2] = 0
    rt[2] = 0
    xt[4, 100] = float("inf")
    xt[5, 7] = float("nan")
    for out in ("f32", "q8", "mxfp8", "f16"):
        y, s, h = ops.rms_norm(xt, w, EPS, residual=rt, out=out)
        if out == "f32":
            assert (y[2] == 0).all() and y[5].isnan().all() and (y[4, :100] == 0).all() and y[4, 100].isnan()
            keep = [0, 1, 3, 6, 7, 8]
            assert torch.equal(y[keep], clean[keep])
        if out == "q8":
            want = ops.quant_q8(clean)
            k = 2048
            for r in (0, 1, 3, 6, 7, 8):
                assert torch.equal(y[r * k:(r + 1) * k], want[r * k:(r + 1) * k])
    big = ops.rms_norm(xt[:1], w, 1e4, out="f32")[0]
    close(f64(big), _want(xt[:1], None, w, 1e4)[1], 32 * U24 * _want(xt[:1], None, w, 1e4)[1].abs(), "eps")


def test_bf16_rounding_is_one(dev):
    import qmm.ops as ops
    xt, rt, w = _inputs(dev, 40, 1000, "bf16", "bf16")
    y, _, h = ops.rms_norm(xt, w, EPS, residual=rt, out="bf16")
    hw, want = _want(xt, rt, w)
    close(f64(y), want, (U8 + 40 * U24) * want.abs(), "y")
    close(f64(h), hw, (U8 + U24) * hw.abs(), "h")
