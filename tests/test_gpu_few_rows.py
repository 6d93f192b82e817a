"""Products of a few rows with an epilogue on the matrix units (f32 / bf16 / Q8_1 rows), and dense MXFP4 products with one: the
rows of a batch do not depend on each other or on its size, nothing outside y is written, weights at every alignment that is
allowed, rows that end inside a chunk of 256 values, replays of a captured call."""
import numpy as np
import pytest
import torch

from sublayer import U24, Weight, close, f64, glu64, act_tol, q8_values, rows, vec

pytestmark = pytest.mark.gpu

KINDS = [("f32", "q4_0"), ("f32", "q4_k"), ("f32", "q6_k"), ("f32", "mxfp4"), ("f32", "mxfp4s"), ("bf16", "q4_0"), ("bf16", "q4_k"),
         ("bf16", "q6_k"), ("bf16", "mxfp4"), ("bf16", "mxfp4s"), ("q8", "q4_0"), ("q8", "q6_k"), ("q8", "mxfp4s")]


def _call(kind, w, x, n, k, up=None, **kw):
    import qmm.ops as ops
    T = x.shape[0]
    if kind == "q8":
        x, kw = ops.quant_q8(x), dict(kw, tokens=T)
    else:
        x, kw = x.to(torch.float32 if kind == "f32" else torch.bfloat16), dict(kw, q8=False)
    if up is not None:
        return ops.ffn_gate_up(w.fmt, x, w.w, up.w, n, k, ws=w.ws, ws2=up.ws, **kw)
    return ops.linear(w.fmt, x, w.w, n, k, ws=w.ws, **kw)


@pytest.mark.parametrize("kind,fmt", KINDS)
@pytest.mark.parametrize("n,k", [(600, 768), (16416, 256)])
def test_rows_do_not_depend_on_the_batch(dev, kind, fmt, n, k):
    """One to four tiles of 16 tokens, one and two tiles of rows a workgroup: the same bits for a row in every call."""
    rng = np.random.default_rng(n + k)
    w, x, b = Weight(fmt, rng, n, k, dev), rows(rng, (63, k), torch.float32, dev), vec(rng, n, dev)
    full = _call(kind, w, x, n, k, bias=b, act="silu", out_dtype=torch.float32)
    for T in (5, 16, 17, 32, 33):
        assert torch.equal(_call(kind, w, x[:T], n, k, bias=b, act="silu", out_dtype=torch.float32), full[:T]), T
    assert torch.equal(_call(kind, w, x[40:57], n, k, bias=b, act="silu", out_dtype=torch.float32), full[40:57])
    if n > 1000:
        return
    up = Weight(fmt, rng, n, k, dev)
    full = _call(kind, w, x, n, k, up, bias=b, out_dtype=torch.float32)
    for T in (5, 16, 17, 33):
        assert torch.equal(_call(kind, w, x[:T], n, k, up, bias=b, out_dtype=torch.float32), full[:T]), T


@pytest.mark.parametrize("kind,fmt", [c for c in KINDS if c[1] in ("q4_0", "mxfp4", "mxfp4s")])
@pytest.mark.parametrize("k", [64, 192, 320, 2112])
def test_rows_end_inside_a_chunk(dev, kind, fmt, k):
    import qmm.ops as ops
    n, T = 70, 6
    rng = np.random.default_rng(k)
    w, up, x = Weight(fmt, rng, n, k, dev), Weight(fmt, rng, n, k, dev), rows(rng, (T, k), torch.float32, dev)
    xv = {"f32": lambda: f64(x), "bf16": lambda: f64(x.bfloat16()), "q8": lambda: q8_values(ops.quant_q8(x), T, k)}[kind]()
    W, U = torch.from_numpy(w.W), torch.from_numpy(up.W)
    # every product is exact; at most three terms of each are added, and four roundings join a block's
    tol = lambda V: (3 * k + 4) * U24 * (xv.abs() @ V.abs().T) * (9 if fmt == "q4_0" else 1)   # noqa: E731  (dot - 8 S: each within 9 sum |x| d)
    got = f64(_call(kind, w, x, n, k, out_dtype=torch.float32))
    close(got, xv @ W.T, tol(W), "product")
    g, u = xv @ W.T, xv @ U.T
    a = glu64("relu", g, u)
    got = f64(_call(kind, w, x, n, k, up, act="relu", out_dtype=torch.float32))
    close(got, a, tol(W) * (u.abs() + tol(U)) + tol(U) * g.abs() + U24 * a.abs(), "gated")


@pytest.mark.parametrize("kind,fmt", KINDS)
def test_rows_of_nan_and_bytes_outside_y(dev, kind, fmt):
    import qmm.ops as ops
    n, k, T = 130, 512, 19
    rng = np.random.default_rng(9)
    w, x = Weight(fmt, rng, n, k, dev), rows(rng, (T, k), torch.float32, dev)
    want = _call(kind, w, x, n, k, out_dtype=torch.float32)
    for dt in (torch.float32, torch.bfloat16):
        buf = torch.full((T * n + 128,), 3.0, dtype=dt, device=dev)
        _call(kind, w, x, n, k, out_dtype=dt, y=buf[64:64 + T * n].view(T, n))
        assert (buf[:64] == 3).all() and (buf[64 + T * n:] == 3).all()
        assert torch.equal(buf[64:64 + T * n].view(T, n), want.to(dt))
    if kind == "q8":
        return   # Q8_1 codes hold no NaN
    bad = x.clone()
    bad[3] = float("nan")
    bad[17, 5] = float("inf")
    got = _call(kind, w, bad, n, k, out_dtype=torch.float32)
    keep = [i for i in range(T) if i not in (3, 17)]
    assert torch.equal(got[keep], want[keep])
    assert got[3].isnan().all() and not got[17].isfinite().any()


@pytest.mark.parametrize("fmt,offset", [("q4_0", 4), ("q6_k", 4), ("mxfp4", 1), ("q4_k", 16)])
def test_weights_at_the_least_alignment(dev, fmt, offset):
    n, k, T = 50, 512, 7
    rng = np.random.default_rng(10)
    w, x = Weight(fmt, rng, n, k, dev), rows(rng, (T, k), torch.float32, dev)
    want = _call("f32", w, x, n, k, out_dtype=torch.float32)
    flat = w.w.reshape(-1).view(torch.uint8)
    buf = torch.full((flat.numel() + 64,), 255, dtype=torch.uint8, device=dev)
    buf[offset:offset + flat.numel()] = flat
    w.w = buf[offset:offset + flat.numel()]
    assert torch.equal(_call("f32", w, x, n, k, out_dtype=torch.float32), want)


@pytest.mark.parametrize("kind,fmt", [("q8", "q6_k"), ("bf16", "q4_0"), ("f32", "mxfp4")])
def test_replays_on_two_streams(dev, kind, fmt):
    n, k, T = 200, 768, 18
    rng = np.random.default_rng(11)
    w, up, b = Weight(fmt, rng, n, k, dev), Weight(fmt, rng, n, k, dev), vec(rng, n, dev)
    xs = [rows(rng, (T, k), torch.float32, dev) for _ in range(3)]
    call = lambda x: (_call(kind, w, x, n, k, bias=b), _call(kind, w, x, n, k, up, bias=b))   # noqa: E731
    want = [call(x) for x in xs]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        x, g = xs[0].clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = call(x)
        graphs.append((g, x, y))
    side = torch.cuda.Stream()
    for i in (1, 2, 0, 2):
        for j, (g, x, _) in enumerate(graphs):
            x.copy_(xs[(i + j) % 3])
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for j, (_, _, y) in enumerate(graphs):
            assert all(torch.equal(p, q) for p, q in zip(y, want[(i + j) % 3]))
        assert all(torch.equal(p, q) for p, q in zip(call(xs[i]), want[i]))


# MXFP8 rows: one and two column blocks a wave, one row tile to more than a group of them, ragged rows and columns
@pytest.mark.parametrize("fmt,T,n,k", [("mxfp4t", 1, 96, 64), ("mxfp4t", 65, 1056, 4096), ("mxfp4t", 2011, 4128, 192), ("mxfp4t", 850, 9440, 128),
                                       ("mxfp4s", 65, 1000, 4096), ("mxfp4s", 900, 257, 320), ("mxfp4t", 4161, 32, 64)])
def test_mxfp8_rows_have_the_plain_products_bits(dev, fmt, T, n, k):
    import qmm.ops as ops
    rng = np.random.default_rng(T + n)
    w, b = Weight(fmt, rng, n, k, dev), vec(rng, n, dev)
    c, s = ops.quant_mxfp8(rows(rng, (T, k), torch.float32, dev))
    res = rows(rng, (T, n), torch.bfloat16, dev)
    y0 = ops.gemm(fmt, "store", c, w.w, n, k, scales=s, ws=w.ws)
    buf = torch.full((T * n + 64,), 3.0, device=dev)
    ops.linear(fmt, c, w.w, n, k, ws=w.ws, scales=s, bias=b, residual=res, y=buf[:T * n].view(T, n))
    assert torch.equal(buf[:T * n].view(T, n), (y0 + b) + res.float()) and (buf[T * n:] == 3).all()
    for at, out in ((1, torch.float32), (2, torch.bfloat16), (8, torch.bfloat16)):   # y rows that are not on 16 bytes, and some that are
        buf = torch.full((T * n + 64,), 3.0, dtype=out, device=dev)
        got = ops.linear(fmt, c, w.w, n, k, ws=w.ws, scales=s, bias=b, residual=res, y=buf[at:at + T * n].view(T, n))
        assert torch.equal(got, ((y0 + b) + res.float()).to(out)) and (buf[:at] == 3).all() and (buf[at + T * n:] == 3).all()
    g = ops.ffn_gate_up(fmt, c, w.w, w.w, n, k, ws=w.ws, ws2=w.ws, scales=s, bias=b, act="gelu", out_dtype=torch.float32)
    pre, up = f64(y0 + b), f64(y0)
    a = glu64("gelu", pre, up)
    close(f64(g), a, act_tol("gelu", pre, glu64("gelu", pre, torch.ones_like(pre))) * up.abs() + 2 * U24 * a.abs(), "gated")
