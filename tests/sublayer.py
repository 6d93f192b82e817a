"""Inputs and 64-bit references of the feed-forward sub-layer's operator tests (norm, linear with an epilogue, gated block)."""
import math

import numpy as np
import torch

from oracle import formats as of
from oracle import ref
from qmm import synth

U24, U11, U8 = 2.0 ** -24, 2.0 ** -11, 2.0 ** -8     # half a step of f32, f16, bf16, relative to the value

ACTS = ("none", "relu", "silu", "sigmoid", "gelu", "gelu_erf")


class Weight:
    """Random weights of one format: device tensors w / ws, exact values W (f64) and the values staged to f16, W16 (f64)."""

    def __init__(self, fmt, rng, n, k, dev):
        import qmm.ops as ops
        base = {"q4_kt": "q4_k", "q4_0t": "q4_0", "mxfp4s": "mxfp4", "mxfp4t": "mxfp4"}.get(fmt, fmt)
        raw = synth.weights(base, rng, n, k)
        self.fmt, self.ws = fmt, None
        t = torch.from_numpy(np.ascontiguousarray(raw).view(np.uint8).reshape(-1).copy()).to(dev)
        if fmt == "q4_kt":
            self.w = ops.tile_q4k(t, n, k)
        elif fmt == "q4_0t":
            self.w = ops.tile_q40(t, n, k)
        elif fmt in ("mxfp4s", "mxfp4t"):
            self.w, self.ws = ops.repack_mxfp4(t, n, k)
            if fmt == "mxfp4t":
                self.w, self.ws = ops.tile_mxfp4(self.w, self.ws, n, k)
        else:
            self.w = t
        self.W = of.dequantize(base, raw, n, k).astype(np.float64)
        self.W16 = staged(base, raw, n, k)


def staged(fmt, raw, n, k):
    """The weights as the f16 GEMMs stage them, each rounding to f16 in its place."""
    f16 = lambda v: v.astype(np.float16).astype(np.float64)   # noqa: E731
    if fmt == "q4_k":
        d, dmin, sc, m, q = of.q4_k_fields(raw)
        ds = f16(d[:, None].astype(np.float64) * sc)
        mn = f16(-(dmin[:, None].astype(np.float64) * m))
        return f16(q * ds[..., None] + mn[..., None]).reshape(n, k)
    if fmt == "q6_k":
        d, sc, q = of.q6_k_fields(raw)
        ds = f16(d[:, None].astype(np.float64) * sc)
        return f16(np.repeat(ds, 16, 1) * (q - 32)).reshape(n, k)
    if fmt == "q4_0":
        return f16(of.dequant_q4_0(raw, n, k).astype(np.float64))
    return None


def rows(rng, shape, dtype, dev, scale=1.0):
    return torch.from_numpy((scale * rng.standard_normal(shape)).astype(np.float32)).to(dtype).to(dev)


def vec(rng, n, dev, scale=0.5):
    return torch.from_numpy((scale * rng.standard_normal(n)).astype(np.float32)).to(dev)


def f64(t):
    return None if t is None else t.detach().double().cpu()


def act64(name, v):
    """act(v) in 64 bits."""
    if name == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "sigmoid":
        return torch.sigmoid(v)
    if name == "gelu":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    if name == "gelu_erf":
        return 0.5 * v * torch.erfc(-v / math.sqrt(2))
    return v


def glu64(name, g, u):
    if name == "swiglu_oai":
        x = g.clamp(max=7.0)
        return x * torch.sigmoid(1.702 * x) * (u.clamp(-7.0, 7.0) + 1)
    return act64(name, g) * u


def act_tol(name, v, a):
    """Bound on |act32(v) - act(v)| for an exact f32 v (f64 tensors v, a = act(v)). Each function is a few f32 operations and
    library calls of at most 16 half steps together; expf and erfcf also see their argument's rounding: a half step of z
    (times the operations that make it, at most 6) changes e^z by |z| half steps, and erfc(t) by less than 2 t^2 + 2. Past
    v = -88.7 e^-v is infinite in f32 and the result 0: |v e^v| is below 2^-121 there."""
    n = torch.full_like(v, 16.0)
    if name == "gelu":
        n = n + 6 * (2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)).abs().clamp(max=110)
    if name == "gelu_erf":
        n = n + 2 * (v ** 2 + 2)
    if name in ("none", "relu"):
        n = torch.zeros_like(v)
    return n * U24 * a.abs() + (0.0 if name in ("none", "relu") else 2.0 ** -121)


def close(got, want, tol, what):
    """|got - want| <= tol elementwise (f64 tensors)."""
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values off, first at " \
                          f"{bad.nonzero()[0].tolist()}: {got[bad][0]:.9g} for {want[bad][0]:.9g}, tolerance {tol[bad][0]:.3g}"


def q8_values(xq, T, k):
    """The values of a planar Q8_1 buffer in 64 bits."""
    codes = xq[:T * k].view(torch.int8).double().cpu().reshape(T, k // 32, 32)
    d = xq[T * k:].view(torch.float32).double().cpu().reshape(T, k // 32, 2)[..., :1]
    return (codes * d).reshape(T, k)


def mxfp8_values(codes, scales):
    T, k = codes.shape
    v = torch.from_numpy(ref.e4m3_decode(codes.cpu().numpy())).reshape(T, k // 32, 32)
    return (v * torch.exp2(scales.double().cpu() - 127)[..., None]).reshape(T, k)
