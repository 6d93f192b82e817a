"""What the feed-forward sub-layer's operators refuse, without a device: the C entry points' statuses and the errors of the
Python surface. Nothing is launched."""
import ctypes

import pytest
import torch

from test_abi import header_enum, lib  # noqa: F401  (fixture)

F32, F16, BF16, MXFP8, Q8 = 0, 1, 2, 3, 4
NONE = 2


def at(a=0x10000):
    return ctypes.c_void_p(a)


def test_rms_norm_statuses(lib):   # noqa: F811
    st = header_enum("qmm_status")

    def call(rows=4, k=64, x=at(), xd=BF16, r=None, rd=BF16, w=at(), wd=F32, eps=1e-6, h=None, od=BF16, o=at(), s=None):
        return lib.qmm_rms_norm(rows, k, x, xd, r, rd, w, wd, ctypes.c_float(eps), h, od, o, s, None)

    for bad in (dict(x=None), dict(w=None), dict(o=None), dict(h=at()), dict(od=F16), dict(od=MXFP8)):
        assert call(**bad) == st["QMM_ERR_NULL"], bad
    for bad in (dict(xd=F16), dict(xd=Q8), dict(wd=F16), dict(r=at(), rd=F16), dict(od=5), dict(od=-1)):
        assert call(**bad) == st["QMM_ERR_DTYPE"], bad
    for bad in (dict(eps=-1e-6), dict(eps=float("nan"))):
        assert call(**bad) == st["QMM_ERR_RANGE"], bad
    for bad in (dict(rows=0), dict(rows=-1), dict(rows=(1 << 24) + 1), dict(k=0), dict(k=-8), dict(k=32769), dict(k=40, od=Q8),
                dict(k=40, od=MXFP8, s=at())):
        assert call(**bad) == st["QMM_ERR_SHAPE"], bad
    for bad in (dict(x=at(0x10001)), dict(xd=F32, x=at(0x10002)), dict(w=at(0x10002)), dict(r=at(0x10001)), dict(od=Q8, x=at(0x10008)),
                dict(od=Q8, o=at(0x10008)), dict(od=MXFP8, s=at(), w=at(0x10004)), dict(od=F16, s=at(0x10004)),
                dict(r=at(), h=at(0x10001))):
        assert call(**bad) == st["QMM_ERR_ALIGN"], bad


def test_rms_norm_grad_statuses(lib):   # noqa: F811
    st = header_enum("qmm_status")

    def call(rows=4, k=64, h=at(), hd=BF16, w=at(), wd=F32, eps=1e-6, dy=at(), yd=BF16, r=None, rd=BF16, o=at(), od=F32, dw=None, ws=None, wb=0):
        return lib.qmm_rms_norm_grad(rows, k, h, hd, w, wd, ctypes.c_float(eps), dy, yd, r, rd, o, od, dw, ws, wb, None)

    for bad in (dict(h=None), dict(w=None), dict(dy=None), dict(o=None)):
        assert call(**bad) == st["QMM_ERR_NULL"], bad
    for bad in (dict(hd=F16), dict(wd=F16), dict(yd=Q8), dict(od=F16), dict(r=at(), rd=F16), dict(od=-1)):
        assert call(**bad) == st["QMM_ERR_DTYPE"], bad
    assert call(eps=-1.0) == st["QMM_ERR_RANGE"] and call(eps=float("nan")) == st["QMM_ERR_RANGE"]
    for bad in (dict(rows=0), dict(rows=(1 << 24) + 1), dict(k=0), dict(k=32769)):
        assert call(**bad) == st["QMM_ERR_SHAPE"], bad
        assert lib.qmm_rms_norm_grad_workspace_size(bad.get("rows", 4), bad.get("k", 64)) == -1
    need = lib.qmm_rms_norm_grad_workspace_size(4, 64)
    assert need > 0
    for bad in (dict(h=at(0x10001)), dict(w=at(0x10002)), dict(dy=at(0x10001)), dict(o=at(0x10002)), dict(r=at(0x10001)), dict(dw=at(0x10002), ws=at(), wb=need),
                dict(dw=at(), ws=at(0x10008), wb=need)):
        assert call(**bad) == st["QMM_ERR_ALIGN"], bad
    for bad in (dict(dw=at()), dict(dw=at(), ws=at(), wb=need - 1)):
        assert call(**bad) == st["QMM_ERR_WORKSPACE"], bad


def test_linear_and_gate_up_statuses(lib):   # noqa: F811
    st = header_enum("qmm_status")

    def linear(fmt=1, act=NONE, t=4, k=512, n=64, x=at(), xd=Q8, s=None, w=at(), ws=None, b=None, r=None, rd=F32, y=at(), yd=F32):
        return lib.qmm_linear(fmt, act, t, k, n, x, xd, s, w, ws, b, r, rd, y, yd, None)

    def gate(fmt=1, act=0, t=4, k=512, n=64, x=at(), xd=Q8, s=None, w=at(), ws=None, w2=at(), ws2=None, b=None, b2=None, y=at(), yd=F32):
        return lib.qmm_ffn_gate_up(fmt, act, t, k, n, x, xd, s, w, ws, w2, ws2, b, b2, y, yd, None)

    def both(status, cases):
        for bad in cases:
            assert linear(**bad) == st[status], bad
            assert gate(**bad) == st[status], bad

    both("QMM_ERR_RANGE", [dict(act=7), dict(act=-1)])
    assert linear(act=1) == st["QMM_ERR_RANGE"]                       # swiglu_oai takes two matrices
    both("QMM_ERR_NULL", [dict(x=None), dict(w=None), dict(y=None), dict(xd=F16, x=None), dict(xd=F32, w=None),
                          dict(fmt=3, xd=Q8), dict(fmt=3, xd=MXFP8, s=at()), dict(fmt=4, xd=MXFP8, ws=at()), dict(fmt=3, xd=F32)])
    for xd in (F32, BF16, Q8, F16):
        assert gate(xd=xd, w2=None) == st["QMM_ERR_NULL"], xd
    assert gate(fmt=4, xd=MXFP8, s=at(), ws=at(), ws2=None) == st["QMM_ERR_NULL"]
    both("QMM_ERR_DTYPE", [dict(xd=5), dict(yd=F16), dict(yd=Q8)])
    assert linear(r=at(), rd=F16) == st["QMM_ERR_DTYPE"]
    both("QMM_ERR_ALIGN", [dict(y=at(0x10002)), dict(y=at(0x10001), yd=BF16), dict(b=at(0x10002)), dict(x=at(0x10008)),
                           dict(w=at(0x10008)), dict(xd=F16, x=at(0x10008)), dict(xd=F16, s=at(0x10002)), dict(xd=F32, w=at(0x10004))])
    assert linear(r=at(0x10002)) == st["QMM_ERR_ALIGN"] and linear(r=at(0x10001), rd=BF16) == st["QMM_ERR_ALIGN"]
    assert gate(b2=at(0x10002)) == st["QMM_ERR_ALIGN"] and gate(w2=at(0x10008)) == st["QMM_ERR_ALIGN"]
    both("QMM_ERR_FORMAT", [dict(fmt=4, xd=Q8), dict(fmt=2, xd=Q8), dict(fmt=9), dict(fmt=2, xd=F16), dict(fmt=7, xd=F16), dict(fmt=5, xd=F32),
                            dict(fmt=1 | (7 << 8), xd=F16), dict(fmt=1, xd=MXFP8, s=at(), ws=at())])
    both("QMM_ERR_SHAPE", [dict(t=0), dict(n=0), dict(k=0), dict(k=300), dict(xd=F16, k=384), dict(xd=F16, t=0), dict(fmt=5, n=24), dict(fmt=5, k=256),
                           dict(fmt=5, xd=F16, n=24), dict(xd=F16, t=1 << 21, k=512), dict(xd=F16, n=1 << 24, k=512), dict(xd=F32, k=300)])
    for call in (linear, gate):
        kw = dict(fmt=4, xd=MXFP8, s=at(), ws=at(), **({"ws2": at()} if call is gate else {}))
        assert call(**kw, n=48) == st["QMM_ERR_SHAPE"] and call(**kw, k=12352) == st["QMM_ERR_SHAPE"]


def test_backward_statuses(lib):   # noqa: F811
    st = header_enum("qmm_status")

    def grad(fmt=1, act=0, t=4, k=512, n=64, x=at(), s=at(), w=at(), w2=at(), b=None, b2=None, dy=at(), dd=F32, o=at()):
        return lib.qmm_ffn_gate_up_grad(fmt, act, t, k, n, x, s, w, w2, b, b2, dy, dd, o, None)

    def operand(t=4, parts=2, n=64, x=at(), xd=BF16, o=at(), s=at()):
        return lib.qmm_grad_operand(t, parts, n, x, xd, o, s, None)

    def gemm_t(fmt=1, t=4, k=512, n=64, x=at(), s=at(), w=at(), w2=at(), y=at(), yd=F32, ws=at(), wb=1 << 40):
        return lib.qmm_gemm_t(fmt, t, k, n, x, s, w, w2, y, yd, ws, wb, None)

    for bad in (dict(x=None), dict(w=None), dict(w2=None), dict(dy=None), dict(o=None)):
        assert grad(**bad) == st["QMM_ERR_NULL"], bad
    for bad in (dict(fmt=2), dict(fmt=3), dict(fmt=4), dict(fmt=7), dict(fmt=1 | (7 << 8))):
        assert grad(**bad) == st["QMM_ERR_FORMAT"] and gemm_t(**bad) == st["QMM_ERR_FORMAT"], bad
        assert lib.qmm_gemm_t_workspace_size(bad["fmt"], 4, 512, 64, 1) == -1
    for bad in (dict(t=0), dict(k=384), dict(n=0), dict(fmt=5, n=24), dict(fmt=5, k=768), dict(t=1 << 24, n=1 << 20)):
        assert gemm_t(**bad) == st["QMM_ERR_SHAPE"], bad
        assert lib.qmm_gemm_t_workspace_size(bad.get("fmt", 1), bad.get("t", 4), bad.get("k", 512), bad.get("n", 64), 1) == -1
    for bad in (dict(t=0), dict(k=384), dict(n=0), dict(fmt=5, n=24), dict(fmt=5, k=768)):
        assert grad(**bad) == st["QMM_ERR_SHAPE"], bad
    def lin(fmt=1, act=0, t=4, k=512, n=64, x=at(), s=at(), w=at(), b=None, dy=at(), dd=F32, o=at()):
        return lib.qmm_linear_grad(fmt, act, t, k, n, x, s, w, b, dy, dd, o, None)

    for bad in (dict(x=None), dict(w=None), dict(dy=None), dict(o=None)):
        assert lin(**bad) == st["QMM_ERR_NULL"], bad
    for bad in (dict(act=1), dict(act=7), dict(act=-1)):
        assert lin(**bad) == st["QMM_ERR_RANGE"], bad
    for bad in (dict(fmt=2), dict(fmt=4), dict(fmt=7)):
        assert lin(**bad) == st["QMM_ERR_FORMAT"], bad
    for bad in (dict(t=0), dict(k=384), dict(n=0), dict(fmt=5, n=24)):
        assert lin(**bad) == st["QMM_ERR_SHAPE"], bad
    for bad in (dict(dy=at(0x10002)), dict(dy=at(0x10001), dd=BF16), dict(o=at(0x10001)), dict(b=at(0x10002)), dict(x=at(0x10008)), dict(w=at(0x10008))):
        assert lin(**bad) == st["QMM_ERR_ALIGN"], bad
    assert lin(dd=F16) == st["QMM_ERR_DTYPE"]
    for bad in (dict(x=None), dict(s=None), dict(w=None), dict(y=None)):
        assert gemm_t(**bad) == st["QMM_ERR_NULL"], bad
    for bad in (dict(x=None), dict(o=None), dict(s=None)):
        assert operand(**bad) == st["QMM_ERR_NULL"], bad
    assert grad(act=7) == st["QMM_ERR_RANGE"] and operand(parts=3) == st["QMM_ERR_RANGE"] and operand(parts=0) == st["QMM_ERR_RANGE"]
    assert grad(dd=F16) == st["QMM_ERR_DTYPE"] and operand(xd=F16) == st["QMM_ERR_DTYPE"] and gemm_t(yd=F16) == st["QMM_ERR_DTYPE"]
    assert operand(t=0) == st["QMM_ERR_SHAPE"] and operand(n=0) == st["QMM_ERR_SHAPE"]
    for bad in (dict(dy=at(0x10002)), dict(dy=at(0x10001), dd=BF16), dict(o=at(0x10001)), dict(b=at(0x10002)), dict(b2=at(0x10002)), dict(x=at(0x10008)),
                dict(w2=at(0x10008)), dict(s=at(0x10002))):
        assert grad(**bad) == st["QMM_ERR_ALIGN"], bad
    for bad in (dict(x=at(0x10008)), dict(w=at(0x10008)), dict(y=at(0x10002)), dict(y=at(0x10001), yd=BF16), dict(fmt=6, w=at(0x10002))):
        assert gemm_t(**bad) == st["QMM_ERR_ALIGN"], bad
    assert operand(o=at(0x10008)) == st["QMM_ERR_ALIGN"] and operand(x=at(0x10002), xd=F32) == st["QMM_ERR_ALIGN"]
    # few output tiles: parts of the sum in the workspace
    need = lib.qmm_gemm_t_workspace_size(1, 64, 512, 4096, 1)
    assert need > 0 and need % (64 * 512 * 4) == 0
    assert gemm_t(t=64, n=4096, wb=need - 1) == st["QMM_ERR_WORKSPACE"] and gemm_t(t=64, n=4096, ws=None) == st["QMM_ERR_WORKSPACE"]
    assert gemm_t(t=64, n=4096, ws=at(0x10008), wb=need) == st["QMM_ERR_ALIGN"]
    assert lib.qmm_gemm_t_workspace_size(1, 4096, 4096, 512, 0) == 0


@pytest.fixture
def ops(monkeypatch):
    """The op surface on host tensors: its device check passes them and a call that reaches the library fails the test."""
    from qmm import ops as o
    monkeypatch.setattr(o, "_here", lambda *ts: None)

    def reached(name, *args):
        raise AssertionError(f"{name} was reached")
    monkeypatch.setattr(o._lib, "call", reached)
    return o


def test_rms_norm_errors(ops):
    x, w = torch.zeros(4, 64), torch.zeros(64)
    for a, kw in (((torch.zeros(64), w), {}), ((torch.zeros(2, 2, 64), w), {}), ((x.half(), w), {}), ((x, w[:32]), {}), ((x, w.half()), {}),
                  ((x, w), dict(residual=torch.zeros(4, 32))), ((x, w), dict(residual=x.half())), ((x, w), dict(h=x)),
                  ((x, w), dict(residual=x.bfloat16(), h=x)), ((x, w), dict(out="int8")), ((x, w), dict(out=None))):
        with pytest.raises(ValueError):
            ops.rms_norm(*a, **kw)


def test_y_is_not_the_rows_of_x(ops):
    k = 512
    w, x = torch.zeros(k * k // 256 * 144, dtype=torch.uint8), torch.zeros(4, k)
    for call in (lambda: ops.linear("q4_k", x, w, k, k, y=x, act="silu", q8=False), lambda: ops.ffn_gate_up("q4_k", x, w, w, k, k, y=x, q8=False),
                 lambda: ops.gemm_t("q4_k", x, w, k, k, y=x)):
        with pytest.raises(ValueError, match="overlaps"):
            call()


def test_linear_backward_errors(ops):
    n, k, T = 32, 512, 4
    w, x, dy = torch.zeros(n * k // 256 * 144, dtype=torch.uint8), torch.zeros(T, k), torch.zeros(T, n)
    for fmt, xx, d, kw in (("mxfp4s", x, dy, {}), ("q4_k", x, dy, dict(act="swiglu_oai")), ("q4_k", x[:, :256], dy, {}), ("q4_k", x, dy[:2], {}), ("q4_k", x, dy.half(), {}),
                           ("q4_k", x, dy, dict(bias=torch.zeros(8))), ("q4_k", x, dy, dict(scales=torch.zeros(T, 2))), ("q4_k", x.half(), dy, {}),
                           ("q4_k", x.double(), dy, {}), ("q6_k", x, dy, {}), ("q4_k", x.half(), dy, dict(scales=torch.zeros(T, 3)))):
        with pytest.raises(ValueError):
            ops.linear_backward(fmt, xx, w, d, n, k, **kw)


def test_rms_norm_backward_errors(ops):
    x, w = torch.zeros(4, 64), torch.zeros(64)
    for a, kw in (((torch.zeros(64), w, x), {}), ((x.half(), w, x), {}), ((x, w[:32], x), {}), ((x, w.half(), x), {}), ((x, w, x[:2]), {}), ((x, w, x.half()), {}),
                  ((x, w, x), dict(dh=x[:, :32])), ((x, w, x), dict(dh=x.half())), ((x, w, x), dict(out_dtype=torch.float16)), ((x, w, x), dict(dx=x[:2])),
                  ((x, w, x), dict(dx=x.half())), ((x, w, torch.zeros(4, 64)), dict(dx=x)), ((torch.zeros(4, 64), w, x), dict(dx=x)), ((x, w, x), dict(dx=torch.zeros(4, 64), out_dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            ops.rms_norm_backward(*a, **kw)


def test_linear_errors(ops):
    n, k, T = 32, 512, 4
    w = torch.zeros(n * k // 256 * 144, dtype=torch.uint8)
    x, xq = torch.zeros(T, k), torch.zeros(ops.q8_bytes(T, k), dtype=torch.uint8)
    b, r = torch.zeros(n), torch.zeros(T, n)
    for fmt, xx, kw in (("q4_k", x, dict(act="tanh")), ("q4_k", x, dict(act="swiglu_oai")), ("q4_k", x, dict(bias=b[:8])), ("q4_k", x, dict(bias=b.bfloat16())),
                        ("q4_k", x, dict(residual=r[:2])), ("q4_k", x, dict(residual=r.half())), ("q4_k", x, dict(out_dtype=torch.float16)),
                        ("q4_k", x, dict(bias=b, y=r.half())), ("q4_k", x, dict(bias=b, y=r, out_dtype=torch.bfloat16)), ("q4_k", x, dict(bias=b, y=r[:2])),
                        ("q4_k", x, dict(bias=b, mode="acc", y=r)), ("q4_k", x, dict(bias=b, mode="swiglu", w2=w)), ("q4_k", x, dict(bias=b, w2=w)),
                        ("q4_k", xq, dict(bias=b)), ("q4_k", xq, dict(tokens=T + 1)), ("q4_k", xq, dict(tokens=T - 1)), ("q4_k", xq, dict(tokens=T, scales=r)),
                        ("q4_k", x, dict(tokens=T)), ("q4_k", x, dict(scales=torch.zeros(T, 2))), ("q4_k", x.half(), dict(scales=torch.zeros(T, 3))),
                        ("q4_k", x.half(), dict(scales=torch.zeros(T, 2).double())), ("q4_k", x[:, :256], dict(bias=b)), ("q4_k", x[0], dict(bias=b)),
                        ("q4_k", x.double(), dict(bias=b)), ("mxfp4", torch.zeros(64, k), dict(bias=b, )), ("mxfp4s", x, dict(bias=b)),
                        ("q4_k", x, dict(bias=b, ws=w)), ("q6_k", x, dict(bias=b)), ("q4_0t", torch.zeros(64, k), dict(bias=b))):
        with pytest.raises(ValueError):
            ops.linear(fmt, xx, w, n, k, **kw)
    with pytest.raises(ValueError, match="too small"):
        ops.linear("q4_k", x, w[:-1], n, k, bias=b)
    codes, sc = torch.zeros(T, k, dtype=torch.uint8), torch.zeros(T, k // 32, dtype=torch.uint8)
    nib, ws = torch.zeros(n, k // 2, dtype=torch.uint8), torch.zeros(n, k // 32, dtype=torch.uint8)
    for kw in (dict(scales=sc[:, :4], ws=ws), dict(scales=sc.float(), ws=ws), dict(scales=sc, ws=ws[:8]), dict(scales=sc), dict(scales=sc, ws=ws, tokens=T)):
        with pytest.raises(ValueError):
            ops.linear("mxfp4s", codes, nib, n, k, **kw)


def test_gate_up_errors(ops):
    n, k, T = 32, 512, 4
    w = torch.zeros(n * k // 256 * 144, dtype=torch.uint8)
    x, b, dy = torch.zeros(T, k), torch.zeros(n), torch.zeros(T, n)
    for kw in (dict(act="tanh"), dict(bias=b[:1]), dict(bias2=b.double()), dict(out_dtype=torch.float16), dict(y=dy.half()), dict(tokens=T), dict(ws=w)):
        with pytest.raises(ValueError):
            ops.ffn_gate_up("q4_k", x, w, w, n, k, **kw)
    for w2 in (w[:-1], None):
        with pytest.raises(ValueError, match="too small"):
            ops.ffn_gate_up("q4_k", x, w, w2, n, k)
    for fmt, xx, d, kw in (("mxfp4s", x, dy, {}), ("q4_k", x, dy[:2], {}), ("q4_k", x, dy.half(), {}), ("q4_k", x.half(), dy, {}),
                           ("q4_k", x, dy, dict(scales=torch.zeros(T, 2))), ("q4_k", x, dy, dict(act="tanh")), ("q4_k", x, dy, dict(bias=b[:1])),
                           ("q4_k", x[:, :256], dy, {}), ("q4_k", x.double(), dy, {}), ("q4_k", x.half(), dy, dict(scales=torch.zeros(T, 1)))):
        with pytest.raises(ValueError):
            ops.ffn_gate_up_backward(fmt, xx, w, w, d, n, k, **kw)
    for fmt, g, kw in (("mxfp4t", dy, {}), ("q4_k", dy[:, :8], {}), ("q4_k", dy, dict(w2=w)), ("q4_k", dy.half(), {}), ("q4_k", dy, dict(out_dtype=torch.float16)),
                       ("q4_k", dy, dict(y=dy)), ("q4_k", torch.zeros(T, 2, n), {}), ("q4_k", torch.zeros(0, n), {})):
        with pytest.raises(ValueError):
            ops.gemm_t(fmt, g, w, n, k, **kw)


def test_host_tensors_are_refused():
    from qmm import ops
    with pytest.raises(ValueError, match="device tensors"):
        ops.rms_norm(torch.zeros(2, 64), torch.zeros(64))
    with pytest.raises(ValueError, match="device tensors"):
        ops.gemm_t("q4_k", torch.zeros(2, 64), torch.zeros(144 * 64, dtype=torch.uint8), 64, 256)
