"""The feed-forward sub-layer as it is run: norm, gated block, down projection into the residual rows, on the operands that
pass between them; alone, twice at once on two streams, and captured into a graph that is replayed on new inputs."""
import numpy as np
import pytest
import torch

from helpers import assert_close_rel_l2
from sublayer import Weight, f64, glu64, rows, vec

pytestmark = pytest.mark.gpu
EPS = 1e-6


class Layer:
    def __init__(self, dev, fmt, down, H, F, seed, biases):
        rng = np.random.default_rng(seed)
        self.H, self.F, self.fmt, self.down_fmt = H, F, fmt, down
        self.norm = 1 + vec(rng, H, dev, 0.1)
        self.gate, self.up, self.down = Weight(fmt, rng, F, H, dev), Weight(fmt, rng, F, H, dev), Weight(down, rng, H, F, dev)
        self.b = [vec(rng, F, dev), vec(rng, F, dev), vec(rng, H, dev)] if biases else [None] * 3

    def __call__(self, x, residual, out, act):
        """(residual + x and the block's output added to it) bf16."""
        import qmm.ops as ops
        T = x.shape[0]
        y, scales, h = ops.rms_norm(x, self.norm, EPS, residual=residual, out=out)
        a = ops.ffn_gate_up(self.fmt, y, self.gate.w, self.up.w, self.F, self.H, ws=self.gate.ws, ws2=self.up.ws, bias=self.b[0],
                            bias2=self.b[1], act=act, scales=scales, tokens=T if out == "q8" else None)
        return ops.linear(self.down_fmt, a, self.down.w, self.H, self.F, ws=self.down.ws, bias=self.b[2], residual=h, y=h)

    def exact(self, x, residual, act):
        h = f64(x) + f64(residual)
        y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS) * f64(self.norm)
        W = lambda w: torch.from_numpy(w.W)   # noqa: E731
        b = [0 if t is None else f64(t) for t in self.b]
        a = glu64(act, y @ W(self.gate).T + b[0], y @ W(self.up).T + b[1])
        return h + a @ W(self.down).T + b[2]


# the 8-bit operands' own rounding: E4M3 2^-4 and Q8_1 2^-8 of a group's largest, both at the norm's output and before the
# down projection: rel-L2 at most 6e-2 (E4M3: 2^-4 / sqrt 3 each, twice) and 2e-2, the f16 path 4e-3 with bf16 rows
@pytest.mark.parametrize("fmt,down,out,T,act,tol", [("q4_k", "q6_k", "q8", 1, "silu", 2e-2), ("q4_kt", "q4_kt", "q8", 5, "gelu", 2e-2),
                                                    ("q4_k", "q6_k", "f16", 130, "gelu", 8e-3), ("q4_0", "q4_0", "f16", 64, "silu", 8e-3),
                                                    ("mxfp4t", "mxfp4t", "mxfp8", 70, "swiglu_oai", 8e-2), ("mxfp4s", "mxfp4s", "mxfp8", 3, "silu", 8e-2)])
def test_sublayer(dev, fmt, down, out, T, act, tol):
    layer = Layer(dev, fmt, down, 512, 1024, 3, biases=fmt != "q4_k")
    rng = np.random.default_rng(T)
    x, r = rows(rng, (T, 512), torch.bfloat16, dev), rows(rng, (T, 512), torch.bfloat16, dev)
    got = layer(x, r, out, act)
    assert_close_rel_l2(f64(got).numpy(), layer.exact(x, r, act).numpy(), tol, f"{fmt} {out}")


@pytest.mark.parametrize("fmt,out,T", [("q4_k", "q8", 1), ("q4_k", "f16", 200), ("mxfp4t", "mxfp8", 66)])
def test_streams_and_graph(dev, fmt, out, T):
    layer = Layer(dev, fmt, fmt, 512, 1024, 4, biases=True)
    rng = np.random.default_rng(T)
    xs = [rows(rng, (T, 512), torch.bfloat16, dev) for _ in range(4)]
    rs = [rows(rng, (T, 512), torch.bfloat16, dev) for _ in range(4)]
    want = [layer(x, r, out, "silu") for x, r in zip(xs, rs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None] * 4
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            got[i] = layer(xs[i], rs[i], out, "silu")
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    x, r = xs[0].clone(), rs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x, r, out, "silu")
    for i in (1, 2, 3, 0, 2):   # replayed on other inputs, with eager calls between
        x.copy_(xs[i])
        r.copy_(rs[i])
        graph.replay()
        assert torch.equal(y, want[i])
        assert torch.equal(layer(xs[(i + 1) % 4], rs[(i + 1) % 4], out, "silu"), want[(i + 1) % 4])


def test_backward_in_a_graph_and_on_streams(dev):
    import qmm.ops as ops
    rng = np.random.default_rng(8)
    T, n, k = 70, 320, 512
    wg, wu = Weight("q4_k", rng, n, k, dev), Weight("q4_k", rng, n, k, dev)
    xs = [rows(rng, (T, k), torch.bfloat16, dev) for _ in range(3)]
    dys = [rows(rng, (T, n), torch.bfloat16, dev, 1e-3) for _ in range(3)]
    call = lambda x, dy: ops.ffn_gate_up_backward("q4_k", x, wg.w, wu.w, dy, n, k)   # noqa: E731
    want = [call(x, dy) for x, dy in zip(xs, dys)]
    torch.cuda.synchronize()
    side, got = torch.cuda.Stream(), []
    for i, (x, dy) in enumerate(zip(xs, dys)):   # each call has its own workspace
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            got.append(call(x, dy))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    x, dy = xs[0].clone(), dys[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(x, dy)
    for i in (1, 2, 0, 1):
        x.copy_(xs[i])
        dy.copy_(dys[i])
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
        call(xs[0], dys[0])
        torch.cuda.synchronize()
