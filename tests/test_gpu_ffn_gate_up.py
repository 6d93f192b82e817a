"""GPU parity of the gated block: forward against the two plain products, bit for bit against the framework's swiglu where that
has the same form; gradients against the 64-bit formulas and against differences; the transposed product against the staged
weights in 64 bits, elementwise.

Tolerances. A GEMM's f32 sum of K products errs by at most K half steps of sum |x w| (e below). The gated output and its
gradients then differ by the functions' slopes times e: |act'| <= 1.13, |act''| <= 1.13 for every activation here (GELU's are
the largest), plus the functions' own error (act_tol) and one rounding of the output."""
import numpy as np
import pytest
import torch

from helpers import assert_close_rel_l2
from sublayer import ACTS, U8, U11, U24, Weight, act64, act_tol, close, f64, glu64, rows, vec
from test_gpu_linear_epilogue import _operand, _product

pytestmark = pytest.mark.gpu

GATES = ACTS + ("swiglu_oai",)
CASES = [("q8", "q4_k", 1, 520, 4096), ("q8", "q4_k", 3, 129, 768), ("q8", "q4_k", 9, 4100, 1280), ("q8", "q4_k", 17, 2056, 8192),
         ("q8", "q6_k", 5, 1000, 768), ("q8", "q4_0", 2, 33, 64), ("q8", "q4_kt", 1, 512, 2048), ("q8", "q4_kt", 4, 48, 4096),
         ("q8", "q4_kt", 33, 1040, 1536), ("q8", "q4_0t", 3, 64, 1024), ("q8", "mxfp4s", 3, 65, 320),
         ("bf16", "q4_k", 2, 77, 768), ("bf16", "q4_0", 5, 130, 640), ("f32", "q6_k", 2, 31, 512), ("bf16", "mxfp4", 4, 50, 2880),
         ("f32", "mxfp4s", 2, 50, 2880), ("bf16", "q4_k", 1, 77, 768), ("f32", "q4_0", 17, 33, 128), ("bf16", "q6_k", 63, 100, 1280),
         ("f32", "q4_k", 16, 100, 256), ("q8", "q6_k", 20, 2050, 512), ("bf16", "mxfp4s", 40, 515, 960), ("f16", "q4_k", 100, 300, 512), ("f16", "q4_k", 333, 2100, 512), ("f16", "q4_k", 1, 77, 768),
         ("f16", "q4_kt", 130, 144, 1024), ("f16", "q6_k", 65, 1030, 768), ("f16", "q4_0", 200, 257, 512),
         ("f16", "q6_k", 70, 96, 4096), ("mxfp8", "mxfp4s", 70, 129, 320), ("mxfp8", "mxfp4t", 3, 96, 2880), ("mxfp8", "mxfp4t", 130, 160, 256)]


def _bounds(xv, w, k):
    """(product, error bound) in 64 bits."""
    W = torch.from_numpy(w)
    return xv @ W.T, k * U24 * (xv.abs() @ W.abs().T)


@pytest.mark.parametrize("kind,fmt,T,n,k", CASES)
def test_forward(dev, kind, fmt, T, n, k):
    import qmm.ops as ops
    rng = np.random.default_rng(T + 5 * n + 11 * k)
    wg, wu = Weight(fmt, rng, n, k, dev), Weight(fmt, rng, n, k, dev)
    x, kw, xv = _operand(kind, rng, T, k, dev)
    if kind == "f16":   # back to unit variance: the activations' bends
        kw["scales"] = kw["scales"] * torch.tensor([1.0, 1e-5], device=dev)
        xv = f64(x) * f64(kw["scales"][:, 1:])
    W = [(v.W16 if kind == "f16" else v.W) for v in (wg, wu)]
    (g, eg), (u, eu) = (_bounds(xv, m, k) for m in W)
    b = [vec(rng, n, dev), vec(rng, n, dev)]
    call = lambda **a: ops.ffn_gate_up(fmt, x, wg.w, wu.w, n, k, ws=wg.ws, ws2=wu.ws, **kw, **a)   # noqa: E731
    for act in GATES:
        for b1, b2 in ((b[0], b[1]), (None, None), (None, b[1])):
            G, U = g + (f64(b1) if b1 is not None else 0), u + (f64(b2) if b2 is not None else 0)
            want = glu64(act, G, U)
            a = act64("silu" if act == "swiglu_oai" else act, G)
            up = U.clamp(-7, 7) + 1 if act == "swiglu_oai" else U
            e1, e2 = eg + U24 * (G.abs() + eg), eu + 2 * U24 * (U.abs() + eu + 1)
            tol = 1.13 * e1 * (up.abs() + e2) + e2 * (a.abs() + 1) + 2 * act_tol("silu" if act == "swiglu_oai" else act, G, a) * up.abs() \
                + (8 if kind != "mxfp8" else 40) * U24 * want.abs() + 2.0 ** -120
            got = call(act=act, bias=b1, bias2=b2, out_dtype=torch.float32)
            close(f64(got), want, tol, act)
            yb = call(act=act, bias=b1, bias2=b2, out_dtype=torch.bfloat16)
            assert torch.equal(yb, got.bfloat16())
    # the framework's own swiglu, where it has these operands
    got = call(act="silu", out_dtype=torch.float32)
    if kind == "q8" and (fmt in ("q4_k", "q4_kt", "q4_0t") or T == 1):
        assert torch.equal(got, ops.mv_swiglu_q8(fmt, wg.w, wu.w, x, n, k, tokens=T, ws=wg.ws, ws2=wu.ws))
    elif kind == "f16":
        assert torch.equal(got, ops.gemm(fmt, "swiglu", x, wg.w, n, k, w2=wu.w, scales=kw["scales"]))
    elif kind == "mxfp8":   # that epilogue's sigmoid is the approximate one
        want = ops.gemm(fmt, "swiglu", x, wg.w, n, k, w2=wu.w, scales=kw["scales"], ws=wg.ws, ws2=wu.ws)
        assert_close_rel_l2(f64(got).numpy(), f64(want).numpy(), 2e-6, "swiglu")
    elif kind != "q8" and (kind, fmt) != ("bf16", "q6_k") and fmt != "mxfp4s" and T == 1:
        assert torch.equal(got, ops.mv_swiglu(fmt, wg.w, wu.w, x, n, k))


BACK = [("q4_k", 1, 64, 256), ("q4_k", 77, 768, 512), ("q4_k", 130, 333, 768), ("q4_k", 300, 1000, 512), ("q4_kt", 70, 144, 1024),
        ("q6_k", 65, 321, 512), ("q6_k", 3, 7, 256), ("q4_0", 77, 768, 256), ("q4_0", 129, 65, 768), ("q4_kt", 5, 16, 512)]


def _grads64(act, g, u, dy):
    g, u = g.clone().requires_grad_(), u.clone().requires_grad_()
    (glu64(act, g, u) * dy).sum().backward()
    return g.grad if g.grad is not None else torch.zeros_like(g), u.grad


@pytest.mark.parametrize("fmt,T,n,k", BACK)
@pytest.mark.parametrize("act", GATES)
def test_backward(dev, fmt, T, n, k, act):
    import qmm.ops as ops
    rng = np.random.default_rng(T + n + k)
    wg, wu = Weight(fmt, rng, n, k, dev), Weight(fmt, rng, n, k, dev)
    x = rows(rng, (T, k), torch.bfloat16, dev)
    dy = rows(rng, (T, n), torch.bfloat16 if T % 2 else torch.float32, dev, 1e-4)
    b = [vec(rng, n, dev), vec(rng, n, dev)] if n % 2 == 0 else [None, None]
    dx, dgu = ops.ffn_gate_up_backward(fmt, x, wg.w, wu.w, dy, n, k, bias=b[0], bias2=b[1], act=act, out_dtype=torch.float32)
    assert dx.shape == (T, k) and dgu.shape == (T, 2, n) and dgu.dtype == torch.bfloat16
    x16, s = ops.row_scale_f16(x)
    xv = f64(x16) * f64(s[:, 1:])
    (g, eg), (u, eu) = _bounds(xv, wg.W16, k), _bounds(xv, wu.W16, k)
    if b[0] is not None:
        g, u = g + f64(b[0]), u + f64(b[1])
    eg, eu = eg + U24 * g.abs(), eu + U24 * u.abs()
    wantg, wantu = _grads64(act, g, u, f64(dy))
    d = f64(dy).abs()
    up = u.clamp(-7, 7) + 1 if act == "swiglu_oai" else u
    a = act64("silu" if act == "swiglu_oai" else act, g)
    slope_err = 1.13 * eg * (2.0 if act == "swiglu_oai" else 1.0) + 200 * U24   # act'' e, and its own few hundred half steps
    tolg = d * (slope_err * (up.abs() + eu) + 1.13 * eu)
    tolu = d * (1.13 * eg + 2 * act_tol("silu" if act == "swiglu_oai" else act, g, a) + 8 * U24 * a.abs())
    for name, got, want, tol, skip in (("dg", dgu[:, 0], wantg, tolg, {"relu": g.abs() <= eg, "swiglu_oai": (g - 7).abs() <= eg}),
                                       ("du", dgu[:, 1], wantu, tolu, {"swiglu_oai": (u.abs() - 7).abs() <= eu})):
        tol = tol + U8 * (want.abs() + tol) + 2.0 ** -126
        if act in skip:   # on a kink the two sides' slopes are both right
            tol = torch.where(skip[act], torch.full_like(tol, float("inf")), tol)
        close(f64(got), want, tol, name)
    # dx from the dgu the call returned: exact but for the operand's rounding to f16 and the sum
    gt = f64(dgu).reshape(T, 2 * n)
    W = torch.from_numpy(np.concatenate([wg.W16, wu.W16]))
    amax = gt.abs().amax(-1, keepdim=True)
    tol = ((2 * n + 64) * U24) * (gt.abs() @ W.abs()) + 2.0 ** -24 * 2.0 ** -13 * amax * W.abs().sum(0)   # f16 subnormals of a row
    close(f64(dx), gt @ W, tol + 2.0 ** -140, "dx")
    dxb, dgub = ops.ffn_gate_up_backward(fmt, x, wg.w, wu.w, dy, n, k, bias=b[0], bias2=b[1], act=act)
    assert torch.equal(dxb, dx.bfloat16()) and torch.equal(dgub, dgu)
    dx2, _ = ops.ffn_gate_up_backward(fmt, x16, wg.w, wu.w, dy, n, k, scales=s, bias=b[0], bias2=b[1], act=act)
    assert torch.equal(dx2, dxb)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_erf", "sigmoid", "none", "swiglu_oai"])
def test_backward_against_differences(dev, act):
    """<dx, v> against the central difference of the 64-bit forward pass along v, at the staged weights: the difference's own
    error is h^2 |f'''| (h = 1e-4: below 1e-6), dgu's rounding to bf16 is 2^-8 of its terms."""
    import qmm.ops as ops
    rng = np.random.default_rng(11)
    T, n, k = 70, 96, 256
    wg, wu = Weight("q6_k", rng, n, k, dev), Weight("q6_k", rng, n, k, dev)
    x = rows(rng, (T, k), torch.float16, dev)
    s = torch.ones((T, 2), device=dev)
    dy, v = rows(rng, (T, n), torch.float32, dev), rows(rng, (T, k), torch.float32, dev)
    dx, _ = ops.ffn_gate_up_backward("q6_k", x, wg.w, wu.w, dy, n, k, scales=s, act=act, out_dtype=torch.float32)
    Wg, Wu = torch.from_numpy(wg.W16), torch.from_numpy(wu.W16)
    loss = lambda z: (glu64(act, z @ Wg.T, z @ Wu.T) * f64(dy)).sum(-1)   # noqa: E731
    h = 1e-4
    want = (loss(f64(x) + h * f64(v)) - loss(f64(x) - h * f64(v))) / (2 * h)
    dg, du = _grads64(act, f64(x) @ Wg.T, f64(x) @ Wu.T, f64(dy))
    terms = dg.abs() * (f64(v) @ Wg.T).abs() + du.abs() * (f64(v) @ Wu.T).abs()
    close((f64(dx) * f64(v)).sum(-1), want, 1.05 * U8 * terms.sum(-1) + 1e-5 * terms.sum(-1) + 1e-5, act)


@pytest.mark.parametrize("fmt,T,n,k", [("q4_k", 1, 1, 256), ("q4_k", 64, 64, 512), ("q4_k", 65, 63, 512), ("q4_k", 200, 1500, 1024),
                                       ("q4_kt", 33, 208, 512), ("q6_k", 129, 130, 768), ("q4_0", 500, 100, 256), ("q6_k", 40, 4000, 256),
                                       ("q4_k", 130, 300, 8192)])
@pytest.mark.parametrize("two", [False, True])
def test_transposed_product(dev, fmt, T, n, k, two):
    import qmm.ops as ops
    rng = np.random.default_rng(T + n + k)
    w = [Weight(fmt, rng, n, k, dev) for _ in range(1 + two)]
    x = rows(rng, (T, 2, n) if two else (T, n), torch.float32, dev)
    x = x * torch.logspace(-28, 10, T, device=dev).reshape(-1, *([1] * (x.dim() - 1)))   # rows of every size
    if T > 2:
        x[1] = 0
    y = ops.gemm_t(fmt, x, w[0].w, n, k, w2=w[1].w if two else None)
    xv = f64(x).reshape(T, -1)
    W = torch.from_numpy(np.concatenate([m.W16 for m in w]))
    tol = (U11 + (2 * n + 64) * U24) * (xv.abs() @ W.abs()) + U24 * 2.0 ** -13 * xv.abs().amax(-1, keepdim=True) * W.abs().sum(0)
    close(f64(y), xv @ W, tol + 2.0 ** -126, "y")
    if T > 2:
        assert (y[1] == 0).all()
    # twice the same bits, into a given y, and nothing past it
    guard = torch.full((T * k + 32,), 5.0, device=dev)
    y2 = ops.gemm_t(fmt, x, w[0].w, n, k, w2=w[1].w if two else None, y=guard[:T * k].view(T, k))
    assert torch.equal(y2, y) and (guard[T * k:] == 5).all()
    if T > 4:   # infinities and NaN stay in their rows
        x[2].view(-1)[0] = float("nan")
        x[3].view(-1)[0] = float("inf")
        y3 = ops.gemm_t(fmt, x, w[0].w, n, k, w2=w[1].w if two else None)
        keep = [i for i in range(T) if i not in (2, 3)]
        assert torch.equal(y3[keep], y[keep]) and y3[2].isnan().all()


def test_grad_operand(dev):
    """Rows scaled by a power of two to [2^13, 2^14), columns added up to a multiple of 64 zero."""
    import qmm.ops as ops
    from qmm import _lib
    rng = np.random.default_rng(2)
    for parts, n in ((1, 1), (1, 64), (2, 65), (2, 1000)):
        T, N = 6, -(-n // 64) * 64
        x = rows(rng, (T, parts, n), torch.float32, dev) * torch.tensor([1e-40, 1e-25, 1e-3, 1.0, 1e6, 0.0], device=dev).reshape(-1, 1, 1)
        x16 = torch.full((T, parts, N), 9.0, dtype=torch.float16, device=dev)
        s = torch.empty((T, 2), device=dev)
        _lib.call("qmm_grad_operand", T, parts, n, x.data_ptr(), 0, x16.data_ptr(), s.data_ptr(), ops._stream())
        assert (x16[..., n:] == 0).all() and torch.equal(s[:, 0] * s[:, 1], torch.ones(T, device=dev))
        assert torch.equal(x16[..., :n], (x * s[:, :1, None]).half())
        m = (x.abs().amax((1, 2)) * s[:, 0])[1:5]
        assert ((m >= 2.0 ** 13) & (m < 2.0 ** 14)).all() and s[5, 0] == 1


@pytest.mark.parametrize("parts,n,dtype", [(2, 12288, torch.bfloat16), (2, 20000, torch.bfloat16), (1, 32768, torch.float32), (2, 40000, torch.bfloat16),
                                           (2, 264, torch.bfloat16), (2, 2056, torch.float32)])
def test_grad_operand_of_long_rows(dev, parts, n, dtype):
    import qmm.ops as ops
    from qmm import _lib
    T, N = 3, -(-n // 64) * 64
    x = rows(np.random.default_rng(n), (T, parts, n), dtype, dev, 1e-3)
    x[1, parts - 1, n - 1] = 5.0    # a row's largest value is its last
    x[2, 0, 0] = float("nan")
    x16 = torch.full((T, parts, N), 9.0, dtype=torch.float16, device=dev)
    s = torch.empty((T, 2), device=dev)
    _lib.call("qmm_grad_operand", T, parts, n, x.data_ptr(), ops._dt(x), x16.data_ptr(), s.data_ptr(), ops._stream())
    assert (x16[..., n:] == 0).all()
    assert torch.equal(x16[:2, :, :n], (x.float() * s[:, :1, None]).half()[:2])
    assert x16[2, 0, 0].isnan() and x16[2, :, :n].isnan().sum() == 1 and s[1].tolist() == [2.0 ** 11, 2.0 ** -11]
