"""Gradients and gated values where few bits or no bits of the answer are left: the sigmoid's slope far from zero, gradient rows
near the largest floats, arguments that are NaN, rows of padding."""
import numpy as np
import pytest
import torch

from sublayer import U8, U24, Weight, close, f64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [336, 333])
def test_sigmoid_slope_keeps_its_bits(dev, n):
    """s(v) s(-v) elementwise relative to itself from -30 to 30, where 1 - s(v) has none of its bits left (rows of zeros: the bias is
    the argument). e^-|v| by the hardware: its argument and the constant of its product with log2 e are a half step each of |v|,
    so 2 |v| half steps, two for the exponential, two for 1 + e, and twice the reciprocal's two, then three products; one rounding to
    bf16."""
    import qmm.ops as ops
    v = torch.linspace(-30, 30, n)
    w, b, one = Weight("q4_0", np.random.default_rng(1), n, 256, dev), v.to(dev), torch.ones(n, device=dev)
    x, s, dy = torch.zeros((3, 256), dtype=torch.float16, device=dev), torch.ones((3, 2), device=dev), torch.ones((3, n), device=dev)
    want = torch.sigmoid(v.double()) * torch.sigmoid(-v.double())
    tol = (1 + U8) * (2 * v.double().abs() + 11) * U24 * want + U8 * want
    _, dpre = ops.linear_backward("q4_0", x, w.w, dy, n, 256, scales=s, bias=b, act="sigmoid")
    _, dgu = ops.ffn_gate_up_backward("q4_0", x, w.w, w.w, dy, n, 256, scales=s, bias=b, bias2=one, act="sigmoid")
    close(f64(dpre), want.expand(3, n), tol.expand(3, n), "dpre")
    close(f64(dgu[:, 0]), want.expand(3, n), tol.expand(3, n), "dg")


@pytest.mark.parametrize("n", [64, 63, 8 * 8193])
def test_gradient_rows_near_the_largest_floats(dev, n):
    """The exponent of a row's scale reaches the largest floats': finite rows stay finite, in [2^13, 2^14) for their largest value."""
    import qmm.ops as ops
    from qmm import _lib
    T, N = 5, -(-n // 64) * 64
    x = torch.from_numpy(np.random.default_rng(2).uniform(-1, 1, (T, 1, n)).astype(np.float32)).to(dev)
    x[:, 0, 0] = 1
    x = x * torch.tensor([2.0 ** 113, 2.0 ** 114, 2.0 ** 117, 2.0 ** 126, 2.0 ** 127], device=dev).reshape(-1, 1, 1)
    x16 = torch.empty((T, 1, N), dtype=torch.float16, device=dev)
    s = torch.empty((T, 2), device=dev)
    _lib.call("qmm_grad_operand", T, 1, n, x.data_ptr(), 0, x16.data_ptr(), s.data_ptr(), ops._stream())
    assert torch.equal(s[:, 1].log2(), torch.tensor([100.0, 101, 104, 113, 114], device=dev)) and (s[:, 0] * s[:, 1] == 1).all()
    assert torch.equal(x16[..., :n], (x * s[:, :1, None]).half()) and (x16[..., n:] == 0).all()
    assert (x16.abs().amax((1, 2)) == 2.0 ** 13).all()


@pytest.mark.parametrize("kind,fmt,T,n,k", [("f16", "q4_k", 70, 96, 256), ("f16", "q6_k", 70, 95, 256), ("f16", "q4_0", 1500, 2104, 256), ("f32", "q4_0", 1, 40, 256),
                                            ("f32", "q4_0", 9, 40, 256), ("q8", "q4_k", 1, 40, 512), ("q8", "q4_k", 20, 40, 512), ("mxfp8", "mxfp4t", 70, 96, 256),
                                            ("mxfp8", "mxfp4s", 70, 95, 256)])
def test_clamped_gate_of_nan_is_nan(dev, kind, fmt, T, n, k):
    """swiglu_oai's clamps keep a NaN of either projection, and take infinities to their limits."""
    import qmm.ops as ops
    from test_gpu_linear_epilogue import _operand
    rng = np.random.default_rng(n)
    w = Weight(fmt, rng, n, k, dev)
    x, kw, _ = _operand(kind, rng, T, k, dev)
    b, b2 = torch.zeros(n, device=dev), torch.zeros(n, device=dev)
    call = lambda: ops.ffn_gate_up(fmt, x, w.w, w.w, n, k, ws=w.ws, ws2=w.ws, bias=b, bias2=b2, act="swiglu_oai", out_dtype=torch.float32, **kw)   # noqa: E731
    clean = call()
    b[3], b2[5] = float("nan"), float("nan")
    b[7], b2[8], b2[9] = float("inf"), float("inf"), float("-inf")
    y = call()
    assert y[:, [3, 5]].isnan().all() and y[:, [7, 8, 9]].isfinite().all()
    keep = [i for i in range(n) if i not in (3, 5, 7, 8, 9)]
    assert torch.equal(y[:, keep], clean[:, keep])
    if kind != "f16":
        return
    dy = torch.ones((T, n), device=dev)
    _, dgu = ops.ffn_gate_up_backward(fmt, x, w.w, w.w, dy, n, k, bias=b, bias2=b2, act="swiglu_oai", **kw)
    assert dgu[:, 0, 3].isnan().all()
    for d in (dgu[:, 1, 3], dgu[:, 0, 5]):   # past a limit its slope is 0 whatever the other's value
        assert (d.isnan() | (d == 0)).all()
    assert dgu[:, 0, 5].isnan().any()


@pytest.mark.parametrize("fmt,T,n,k", [("q4_k", 200, 136, 512), ("q6_k", 200, 133, 512), ("q4_0", 77, 768, 256), ("q4_k", 2011, 4104, 256), ("q4_kt", 1000, 2064, 512),
                                       ("q6_k", 1500, 4099, 256)])
def test_padding_rows_have_no_gradient(dev, fmt, T, n, k):
    """64-row tiles of padding rows: zeros in dpre, dgu and dx, so that sums over the rows (a bias's gradient) hold the others' alone."""
    import qmm.ops as ops
    from qmm import _lib
    from qmm.formats import CODE
    rng = np.random.default_rng(T)
    w, u = Weight(fmt, rng, n, k, dev), Weight(fmt, rng, n, k, dev)
    x = torch.from_numpy(rng.standard_normal((T, k)).astype(np.float32)).to(dev)
    dy = torch.from_numpy(rng.standard_normal((T, n)).astype(np.float32)).to(dev)
    b = torch.from_numpy(rng.standard_normal(n).astype(np.float32)).to(dev)
    live = torch.ones(T, dtype=torch.bool, device=dev)
    live[64:128] = False
    live[64 * ((T - 1) // 64):] = False   # the last tile, ragged
    if T > 1000:
        live[512:1024] = False            # whole tiles of 128 rows and more
    info = live.int().reshape(-1, 1).expand(T, 4).contiguous()
    x16, s = ops.row_scale_f16(x, info=info)
    full, fs = ops.row_scale_f16(x)
    assert (s[~live, 0] == 0).all() and torch.equal(x16[live], full[live])
    dpre = torch.full((T, n), float("nan"), dtype=torch.bfloat16, device=dev)
    dgu = torch.full((T, 2, n), float("nan"), dtype=torch.bfloat16, device=dev)
    st = ops._stream()
    _lib.call("qmm_linear_grad", CODE[fmt], 0, T, k, n, x16.data_ptr(), s.data_ptr(), w.w.data_ptr(), b.data_ptr(), dy.data_ptr(), 0, dpre.data_ptr(), st)
    _lib.call("qmm_ffn_gate_up_grad", CODE[fmt], 0, T, k, n, x16.data_ptr(), s.data_ptr(), w.w.data_ptr(), u.w.data_ptr(), b.data_ptr(), None, dy.data_ptr(), 0,
              dgu.data_ptr(), st)
    dx, dp = ops.linear_backward(fmt, x16, w.w, dy, n, k, scales=s, bias=b, act="silu")
    dx2, dg = ops.ffn_gate_up_backward(fmt, x16, w.w, u.w, dy, n, k, scales=s, bias=b)
    want = ops.linear_backward(fmt, full, w.w, dy, n, k, scales=fs, bias=b, act="silu")
    want2 = ops.ffn_gate_up_backward(fmt, full, w.w, u.w, dy, n, k, scales=fs, bias=b)
    for got, ref in ((dpre, want[1]), (dgu, want2[1]), (dp, want[1]), (dg, want2[1]), (dx, want[0]), (dx2, want2[0])):
        assert torch.equal(got[live], ref[live]) and (got[~live] == 0).all()


@pytest.mark.parametrize("fmt,T,n,k", [("q4_k", 200, 136, 512), ("q6_k", 200, 133, 512), ("q4_0", 1, 768, 256), ("q4_k", 2011, 4104, 256), ("q4_kt", 1000, 2064, 512),
                                       ("q6_k", 1500, 4099, 256)])
def test_padding_rows_among_others_have_no_gradient(dev, fmt, T, n, k):
    """The same for single padding rows, whose dy holds anything: zero like those of whole tiles, the rows beside them unchanged."""
    import qmm.ops as ops
    rng = np.random.default_rng(T + 1)
    w, u = Weight(fmt, rng, n, k, dev), Weight(fmt, rng, n, k, dev)
    x = torch.from_numpy(rng.standard_normal((T, k)).astype(np.float32)).to(dev)
    b = torch.from_numpy(rng.standard_normal(n).astype(np.float32)).to(dev)
    live = torch.from_numpy(rng.random(T) < 0.7).to(dev) if T > 1 else torch.zeros(T, dtype=torch.bool, device=dev)
    x16, s = ops.row_scale_f16(x, info=live.int().reshape(-1, 1).expand(T, 4).contiguous())
    full, fs = ops.row_scale_f16(x)
    for dt in (torch.float32, torch.bfloat16):
        clean = torch.from_numpy(rng.standard_normal((T, n)).astype(np.float32)).to(dt).to(dev)
        dy = torch.where(live[:, None], clean, torch.full_like(clean, float("nan")))
        got = ops.linear_backward(fmt, x16, w.w, dy, n, k, scales=s, bias=b, act="gelu") + \
            ops.ffn_gate_up_backward(fmt, x16, w.w, u.w, dy, n, k, scales=s, bias=b, bias2=b)
        want = ops.linear_backward(fmt, full, w.w, clean, n, k, scales=fs, bias=b, act="gelu") + \
            ops.ffn_gate_up_backward(fmt, full, w.w, u.w, clean, n, k, scales=fs, bias=b, bias2=b)
        for g, r in zip(got, want):
            assert torch.equal(g[live], r[live]) and (g[~live] == 0).all()
