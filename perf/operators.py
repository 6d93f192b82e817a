"""The measured calls of the dense feed-forward sub-layer on quantized weights, through ``qmm.ops``.

    rms_norm              h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight, written as the operand that the next
                          product reads: Q8_1, MXFP8, row-scaled f16, or plain bf16 / f32 rows
    linear                y = act(x W^T + bias) + residual on quantized W
    ffn_gate_up           y = act(x Wg^T + bg) (x Wu^T + bu)
    ffn_gate_up_backward  dgu = (dL/d(x Wg^T + bg), dL/d(x Wu^T + bu)) and dx = dg Wg + du Wu (frozen quantized weights:
                          what an adapter below or beside the projections trains on)

The listed cases are these calls at the sizes of this repository's dense layers (hidden 4096, FFN 12288) and expert
layers (2048 / 768, 2880 / 2880), from one decoded token to prompts and training batches of thousands; ``draw`` takes any
format, operand, activation and size of the same ranges.

Weights have a trained layer's magnitudes (outputs of order one); activations are rows of unit variance. Where a call
takes an 8-bit operand, the operand is the input. ``own`` False computes the plain form in 32 bits.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6
BLOCK = {"q4_0": (32, 18), "q4_k": (256, 144), "q6_k": (256, 210), "mxfp4s": (32, 17)}   # values, bytes
PLAIN = {"q4_kt": "q4_k", "mxfp4t": "mxfp4s"}                                            # what a tiled copy is made from
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
ACTS = ("none", "relu", "silu", "sigmoid", "gelu", "gelu_erf")
TYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def _ops():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "loom-skills_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from qmm import ops
    return ops


def _norm(name, rows, k, x, residual, out):
    return {"name": name, "kind": "norm", "rows": rows, "k": k, "x": x, "residual": residual, "out": out}


def _product(kind, name, fmt, tokens, n, k, x, bias, act, residual, out):
    return {"name": name, "kind": kind, "fmt": fmt, "tokens": tokens, "n": n, "k": k, "x": x, "bias": bias, "act": act,
            "residual": residual, "out": out}


def listed():
    return [
        # one decoded token before its projections: the residual's addition, and the int8 matvecs' operand
        _norm("norm 1 x 4096 to q8", 1, 4096, "bf16", True, "q8"),
        # a ragged prompt chunk before MXFP4 projections
        _norm("norm 333 x 2880 to mxfp8", 333, 2880, "f32", True, "mxfp8"),
        # the per-head norm of a prompt's queries: many short rows
        _norm("norm 65536 x 128 to bf16", 65536, 128, "bf16", False, "bf16"),
        # a long prompt before the f16 GEMMs
        _norm("norm 4096 x 4096 to f16", 4096, 4096, "bf16", True, "f16"),
        # an output projection of one decoded token into the residual rows
        _product("linear", "linear q4_k 1 token", "q4_k", 1, 4096, 4096, "q8", True, "none", True, "bf16"),
        # a few drafted tokens on f32 rows through a projection with an activation
        _product("linear", "linear q4_0 5 tokens gelu", "q4_0", 5, 6144, 2048, "f32", True, "gelu", False, "f32"),
        # a ragged prompt through the down projection into the residual rows
        _product("linear", "linear q6_k 333 tokens", "q6_k", 333, 4096, 12288, "f16", False, "none", True, "bf16"),
        # a long prompt through an MXFP4 projection with its bias, into the residual rows
        _product("linear", "linear mxfp4t 4096 tokens", "mxfp4t", 4096, 2880, 2880, "mxfp8", True, "none", True, "bf16"),
        # gate and up of one decoded token: the largest weight stream of a decode step
        _product("gate_up", "gate_up q4_kt 1 token", "q4_kt", 1, 12288, 4096, "q8", False, "silu", False, "f32"),
        # gate and up of a ragged prompt, GELU-gated, with biases
        _product("gate_up", "gate_up q4_k 700 tokens gelu", "q4_k", 700, 12288, 4096, "f16", True, "gelu", False, "bf16"),
        # the gradients of a small block for a short batch
        _product("grad", "gate_up grad q4_0 77 tokens", "q4_0", 77, 768, 2048, "f16", True, "silu", False, "bf16"),
        # the gradients of a dense layer's block for a training batch
        _product("grad", "gate_up grad q4_k 2048 tokens", "q4_k", 2048, 12288, 4096, "f16", False, "silu", False, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "linear", "linear", "gate_up", "grad"])
    if kind == "norm":
        out = rng.choice(["q8", "mxfp8", "f16", "bf16", "f32"])
        k = 32 * _log_int(rng, 1, 400) if out in ("q8", "mxfp8") else _log_int(rng, 1, 12800)
        c = _norm("", min(_log_int(rng, 1, 65536), (1 << 24) // k), k, rng.choice(["bf16", "f32"]), rng.random() < 0.6, out)
    else:
        x = "f16" if kind == "grad" else rng.choice(["q8", "q8", "f16", "f16", "mxfp8", "bf16", "f32"])
        fmt = rng.choice({"q8": ["q4_k", "q4_kt", "q6_k", "q4_0", "mxfp4s"], "f16": ["q4_k", "q4_kt", "q6_k", "q4_0"],
                          "mxfp8": ["mxfp4s", "mxfp4t"]}.get(x, ["q4_k", "q6_k", "q4_0", "mxfp4s"]))
        tokens = _log_int(rng, 64, 4096) if x in ("f16", "mxfp8") else _log_int(rng, 1, 63)
        if kind == "grad":
            tokens = _log_int(rng, 1, 2048)
        k = 512 * _log_int(rng, 1, 24)
        if fmt == "q4_kt" and x == "q8":                        # the tiled matvec: at most 8 waves of at most 4 units
            k = 512 * rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 15, 16, 18, 20, 21, 24])
        n = _log_int(rng, 256, 12288)                           # GGUF rows: any count
        n = n if fmt in ("q4_k", "q6_k", "q4_0") else n // 32 * 32
        tokens = max(1, min(tokens, int(8.2e11 / (n * k * {"linear": 2, "gate_up": 4, "grad": 8}[kind]))))
        out = "bf16" if x in ("f16", "mxfp8") else rng.choice(["bf16", "f32"])
        # no gradient of relu: its slope jumps at 0, where the two sides' sums differ in their last bits
        act = rng.choice([a for a in ACTS if kind != "grad" or a != "relu"])
        c = _product(kind, "", fmt, tokens, n, k, x, rng.random() < 0.5, act,
                     kind == "linear" and rng.random() < 0.5, out)
    del c["name"]
    return c


# -------------------------------------------------------------------------------------------------------- inputs
def _bytes(g, *shape):
    return torch.randint(0, 256, shape, dtype=torch.uint8, device=DEV, generator=g)


def _f16_bytes(v):
    return v.to(torch.float16).view(torch.uint8).reshape(*v.shape, 2)


def _weight(g, fmt, rows, k):
    """Random weights in a storage format: GGUF block bytes u8 [rows, blocks, bytes], or for mxfp4s the planes (nibbles
    u8 [rows, k / 2], E8M0 u8 [rows, k / 32]). Values of about 1 / sqrt(k)."""
    size = math.sqrt(4096 / k)
    if fmt == "mxfp4s":
        mid = 121 + int(round(math.log2(size)))
        return _bytes(g, rows, k // 2), torch.randint(mid - 2, mid + 2, (rows, k // 32), dtype=torch.uint8, device=DEV, generator=g)
    values, nbytes = BLOCK[fmt]
    nb = k // values
    w = _bytes(g, rows, nb, nbytes)
    u = size * (0.5 + torch.rand((rows, nb), device=DEV, generator=g))
    if fmt == "q4_0":
        w[..., 0:2] = _f16_bytes(3.4e-3 * u)
    elif fmt == "q4_k":                                         # dmin about 7.5 d: the codes are centred on zero
        w[..., 0:2] = _f16_bytes(9e-5 * u)
        w[..., 2:4] = _f16_bytes(6.75e-4 * u)
    else:
        w[..., 208:210] = _f16_bytes(1.1e-5 * u)
    return w


def _stored(fmt, raw, rows, k):
    """(w, ws) as a program keeps them: the bytes, or the tiled copy made once at load time."""
    if fmt == "mxfp4s":
        return raw
    if fmt == "mxfp4t":      # [rows / 32][k / 64][half][32 rows][16 bytes], scales [rows / 32][k / 256][half][32][4]
        c = k // 64
        nib = raw[0].reshape(rows // 32, 32, c, 2, 16).permute(0, 2, 3, 1, 4).contiguous()
        sc = torch.nn.functional.pad(raw[1].reshape(rows // 32, 32, c, 2), (0, 0, 0, -c % 4))
        sc = sc.reshape(rows // 32, 32, -1, 4, 2).permute(0, 2, 4, 1, 3).contiguous()
        return nib.reshape(-1), sc.reshape(-1)
    if fmt == "q4_kt":       # [rows / 16][k / 512]: headers [16][2][16 bytes], then code planes [4][16][2][2][16 bytes]
        b = raw.reshape(rows // 16, 16, k // 512, 2, 144)
        head = b[..., :16].permute(0, 2, 1, 3, 4).reshape(rows // 16, k // 512, 512)
        codes = b[..., 16:].reshape(rows // 16, 16, k // 512, 2, 2, 4, 16).permute(0, 2, 5, 1, 3, 4, 6)
        return torch.cat([head, codes.reshape(rows // 16, k // 512, 4096)], -1).reshape(-1), None
    return raw.reshape(-1), None


def _q8(v):
    """(codes, f16-rounded d) of Q8_1: per 32 values d = amax / 127, codes rounded half away from zero."""
    g = v.reshape(v.shape[0], -1, 32)
    d = g.abs().amax(-1, keepdim=True)
    d = d / torch.full_like(d, 127.0)                           # a division (by a plain number torch multiplies)
    t = torch.where(d > 0, g / d, torch.zeros_like(g))
    return torch.sign(t) * torch.floor(t.abs() + 0.5), d.half()


def _mxfp8(v):
    """(E4M3 codes [rows, k], E8M0 bytes [rows, k / 32]): a power of two per 32 values, the largest below 256."""
    g = v.reshape(v.shape[0], -1, 32)
    a = g.abs().amax(-1, keepdim=True)
    e = torch.where(a > 0, torch.frexp(a)[1] - 8, torch.full_like(a, -127, dtype=torch.int32)).clamp(-127, 127)
    codes = torch.ldexp(g, -e).float().to(torch.float8_e4m3fn)
    return codes.reshape(v.shape), (e + 127).to(torch.uint8).reshape(v.shape[0], -1)


def _operand(kind, x):
    """(operand, scales) of rows x as the calls take them."""
    if kind == "q8":
        q, d = _q8(x)
        meta = torch.stack([d.squeeze(-1).float(), q.sum(-1)], -1)
        return torch.cat([q.to(torch.int8).view(torch.uint8).reshape(-1), meta.reshape(-1).view(torch.uint8)]), None
    if kind == "f16":
        return x.half(), torch.ones((x.shape[0], 2), device=DEV)
    if kind == "mxfp8":
        codes, e = _mxfp8(x)
        return codes.view(torch.uint8), e
    return x.to(TYPE[kind]), None


def prepare(case, seed):
    c, g = case, torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"c": c}
    if c["kind"] == "norm":
        shape = (c["rows"], c["k"])
        s["x"] = torch.randn(shape, device=DEV, generator=g).to(TYPE[c["x"]])
        s["residual"] = 2 * torch.randn(shape, device=DEV, generator=g) if c["residual"] else None
        if c["residual"]:
            s["residual"] = s["residual"].to(TYPE[c["x"]])
        s["weight"] = 1 + 0.2 * torch.randn(c["k"], device=DEV, generator=g)
        return s
    n, k, t, two = c["n"], c["k"], c["tokens"], c["kind"] != "linear"
    s["raw"] = [_weight(g, PLAIN.get(c["fmt"], c["fmt"]), n, k) for _ in range(1 + two)]
    s["w"] = [_stored(c["fmt"], r, n, k) for r in s["raw"]]
    s["x"], s["scales"] = _operand(c["x"], torch.randn((t, k), device=DEV, generator=g))
    s["bias"] = [0.5 * torch.randn(n, device=DEV, generator=g) if c["bias"] else None for _ in range(1 + two)]
    s["residual"] = torch.randn((t, n), device=DEV, generator=g).to(TYPE[c["out"]]) if c["residual"] else None
    if c["kind"] == "grad":
        s["dy"] = (1e-3 * torch.randn((t, n), device=DEV, generator=g)).bfloat16()
    return s


# ----------------------------------------------------------------------------------------------- the plain form
def _half(b):
    return b.contiguous().view(torch.float16).squeeze(-1).float()


def _values(fmt, raw):
    """The weights in 32 bits [rows, k]."""
    if fmt == "mxfp4s":
        lut = torch.tensor(FP4 + tuple(-v for v in FP4), device=DEV)
        q = torch.stack([raw[0] & 15, raw[0] >> 4], -1).reshape(raw[0].shape[0], -1, 32)
        return (lut[q.int()] * torch.exp2(raw[1].float() - 127)[..., None]).reshape(raw[0].shape[0], -1)
    rows = raw.shape[0]
    if fmt == "q4_0":
        q = torch.cat([raw[..., 2:] & 15, raw[..., 2:] >> 4], -1).float() - 8
        return (_half(raw[..., 0:2])[..., None] * q).reshape(rows, -1)
    if fmt == "q4_k":
        a, b, c = raw[..., 4:8], raw[..., 8:12], raw[..., 12:16]
        sc = torch.cat([a & 63, (c & 15) | ((a >> 6) << 4)], -1).float()
        mn = torch.cat([b & 63, (c >> 4) | ((b >> 6) << 4)], -1).float()
        q = raw[..., 16:].reshape(rows, -1, 4, 32)              # pages: low nibbles sub-block 2p, high nibbles 2p + 1
        q = torch.stack([q & 15, q >> 4], 3).reshape(rows, -1, 8, 32).float()
        d, dmin = _half(raw[..., 0:2]), _half(raw[..., 2:4])
        return ((d[..., None] * sc)[..., None] * q - (dmin[..., None] * mn)[..., None]).reshape(rows, -1)
    ql = raw[..., 0:128].reshape(rows, -1, 2, 2, 32)            # q6_k: half, 32-byte run, byte
    qh = raw[..., 128:192].reshape(rows, -1, 2, 1, 32)
    lo = torch.cat([ql & 15, ql >> 4], 3)                       # groups 0..3 of the half
    sh = torch.arange(0, 8, 2, device=DEV, dtype=torch.uint8).reshape(4, 1)
    q = (lo | (((qh >> sh) & 3) << 4)).float() - 32
    sc = raw[..., 192:208].contiguous().view(torch.int8).float().reshape(rows, -1, 2, 4, 2, 1)
    d = _half(raw[..., 208:210])[..., None, None, None, None]
    return (d * sc * q.reshape(rows, -1, 2, 4, 2, 16)).reshape(rows, -1)


def _rows(c, s):
    """The operand's values in 32 bits [tokens, k]."""
    t, k = c["tokens"], c["k"]
    if c["x"] == "q8":
        q = s["x"][:t * k].view(torch.int8).reshape(t, -1, 32).float()
        return (q * s["x"][t * k:].view(torch.float32).reshape(t, -1, 2)[..., :1]).reshape(t, k)
    if c["x"] == "f16":
        return s["x"].float() * s["scales"][:, 1:]
    if c["x"] == "mxfp8":
        q = s["x"].view(torch.float8_e4m3fn).float().reshape(t, -1, 32)
        return (q * torch.exp2(s["scales"].float() - 127)[..., None]).reshape(t, k)
    return s["x"].float()


def _act(name, v):
    if name == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "gelu_erf":
        return 0.5 * v * (1 + torch.erf(v / math.sqrt(2)))
    return v


def _slope(name, v):
    """d act / d v."""
    if name == "relu":
        return (v > 0).to(v.dtype)
    if name in ("silu", "sigmoid"):
        p = 1 / (1 + torch.exp(-v))
        return p * (1 - p) if name == "sigmoid" else p * (1 + v * (1 - p))
    if name == "gelu":
        t = torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v))
        return 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * v * v)
    if name == "gelu_erf":
        return 0.5 * (1 + torch.erf(v / math.sqrt(2))) + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    return torch.ones_like(v)


def _project(x, w, bias):
    y = torch.matmul(x, w.t())
    return y if bias is None else y + bias


def _normed(c, v):
    """The rows v in the form that the case asks for, 8-bit codes as the values they stand for."""
    if c["out"] == "q8":
        q, d = _q8(v)
        return (q * d.to(v.dtype)).reshape(v.shape).half()
    if c["out"] == "mxfp8":
        codes, e = _mxfp8(v)
        return codes, e.view(torch.float8_e8m0fnu)
    if c["out"] == "f16":
        e = (torch.frexp(v.abs().amax(-1, keepdim=True))[1] - 14).clamp(0, 100)
        one = torch.ones_like(v[:, :1])
        return torch.ldexp(v, -e).half(), torch.cat([torch.ldexp(one, -e), torch.ldexp(one, e)], -1).float()
    return v.to(TYPE[c["out"]])


def _plain(s):
    c = s["c"]
    if c["kind"] == "norm":
        h = s["x"].float()
        if c["residual"]:
            h = h + s["residual"].float()
        y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * s["weight"]
        return _normed(c, y), (h.to(s["residual"].dtype) if c["residual"] else None)
    x = _rows(c, s)
    w = [_values(PLAIN.get(c["fmt"], c["fmt"]), r) for r in s["raw"]]
    if c["kind"] == "linear":
        y = _act(c["act"], _project(x, w[0], s["bias"][0]))
        if c["residual"]:
            y = y + s["residual"].float()
        return y.to(TYPE[c["out"]])
    g, u = _project(x, w[0], s["bias"][0]), _project(x, w[1], s["bias"][1])
    if c["kind"] == "gate_up":
        return (_act(c["act"], g) * u).to(TYPE[c["out"]])
    dy = s["dy"].float()
    dg, du = dy * u * _slope(c["act"], g), dy * _act(c["act"], g)
    return (torch.matmul(dg, w[0]) + torch.matmul(du, w[1])).bfloat16(), torch.stack([dg, du], 1).bfloat16()


def run(state):
    s, c = state, state["c"]
    if not own:
        return _plain(s)
    ops = _ops()
    if c["kind"] == "norm":
        y, scales, h = ops.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], out=c["out"])
        if c["out"] == "q8":                                    # the codes as the values they stand for
            rows, k = s["x"].shape
            codes = y[:rows * k].view(torch.int8).view(rows, -1, 32)
            d = y[rows * k:].view(torch.float32).view(rows, -1, 2)[..., :1]
            y = torch.mul(codes, d, out=torch.empty(codes.shape, dtype=torch.float16, device=y.device)).view(rows, k)
        elif c["out"] == "mxfp8":
            y = y.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)
        elif c["out"] == "f16":
            y = y, scales
        return y, h
    n, k, bias = c["n"], c["k"], s["bias"]
    kw = {"scales": s["scales"], "act": c["act"], "bias": bias[0], "out_dtype": TYPE[c["out"]]}
    (w, ws), (w2, ws2) = s["w"][0], s["w"][-1]
    if c["kind"] != "grad":
        kw["tokens"] = c["tokens"] if c["x"] == "q8" else None
        kw["q8"] = False if c["x"] in TYPE else "auto"          # f32 / bf16 rows are multiplied as they are
    if c["kind"] == "linear":
        return ops.linear(c["fmt"], s["x"], w, n, k, ws=ws, residual=s["residual"], **kw)
    if c["kind"] == "gate_up":
        return ops.ffn_gate_up(c["fmt"], s["x"], w, w2, n, k, ws=ws, ws2=ws2, bias2=bias[1], **kw)
    return ops.ffn_gate_up_backward(c["fmt"], s["x"], w, w2, s["dy"], n, k, bias2=bias[1], **kw)


# -------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["kind"] == "norm":
        v, size = c["rows"] * c["k"], 2 if c["x"] == "bf16" else 4
        out = {"q8": 1.25, "mxfp8": 1 + 1 / 32, "f16": 2 + 8 / c["k"], "bf16": 2, "f32": 4}[c["out"]]
        return {"bytes": v * (size * (3 if c["residual"] else 1) + out) + 4 * c["k"],
                "flops": v * (5 if c["residual"] else 4)}
    t, n, k, m = c["tokens"], c["n"], c["k"], 1 if c["kind"] == "linear" else 2
    values, size = BLOCK[PLAIN.get(c["fmt"], c["fmt"])]
    rows_in = {"q8": 1.25, "f16": 2, "mxfp8": 1 + 1 / 32, "bf16": 2, "f32": 4}[c["x"]]
    fixed = m * n * (k // values) * size + t * k * rows_in + (4 * n * m if c["bias"] else 0)
    if c["kind"] == "grad":                                     # dy in, dgu and dx out
        return {"bytes": fixed + 2 * t * n * 3 + 2 * t * k, "flops": 8 * t * n * k}
    return {"bytes": fixed + t * n * (2 if c["out"] == "bf16" else 4) * (2 if c["residual"] else 1), "flops": 2 * m * t * n * k}


# ----------------------------------------------------------------------------------------- the results in 64 bits
def _nibbles(b, dim):
    return torch.cat([b % 16, torch.div(b, 16, rounding_mode="floor")], dim)


def _exact_weight(fmt, raw):
    """The weights in 64 bits, from the formats' definitions."""
    f64 = torch.float64
    if fmt == "mxfp4s":
        code = _nibbles(raw[0].unsqueeze(-1), -1).flatten(1).long()
        mag = torch.tensor(FP4, dtype=f64, device=DEV)[code % 8]
        val = torch.where(code >= 8, -mag, mag)
        return val * torch.ldexp(torch.ones((), dtype=f64, device=DEV), raw[1].int() - 127).repeat_interleave(32, 1)
    rows, nb = raw.shape[:2]

    def half(at):
        return raw[..., at:at + 2].contiguous().view(torch.float16).to(f64)

    if fmt == "q4_0":
        return ((_nibbles(raw[..., 2:].short(), -1).to(f64) - 8) * half(0)).reshape(rows, -1)
    if fmt == "q4_k":
        p = raw[..., 4:16].short()
        sc = torch.cat([p[..., 0:4] % 64, p[..., 8:12] % 16 + 16 * (p[..., 0:4] // 64)], -1).to(f64)
        mn = torch.cat([p[..., 4:8] % 64, p[..., 8:12] // 16 + 16 * (p[..., 4:8] // 64)], -1).to(f64)
        q = _nibbles(raw[..., 16:].short().reshape(rows, nb, 4, 1, 32), 3).to(f64).reshape(rows, nb, 8, 32)
        return (q * (half(0) * sc)[..., None] - (half(2) * mn)[..., None]).reshape(rows, -1)
    low = _nibbles(raw[..., 0:128].short().reshape(rows, nb, 2, 1, 2, 32), 3).reshape(rows, nb, 2, 4, 32)
    high = raw[..., 128:192].short().reshape(rows, nb, 2, 1, 32)
    high = torch.cat([high % 4, high // 4 % 4, high // 16 % 4, high // 64], 3)
    q = (low + 16 * high - 32).to(f64).reshape(rows, nb, 16, 16)
    sc = raw[..., 192:208].contiguous().view(torch.int8).to(f64)
    return (q * (sc * half(208))[..., None]).reshape(rows, -1)


def _exact_rows(c, s):
    t, k = c["tokens"], c["k"]
    if c["x"] == "q8":
        pair = s["x"][t * k:].view(torch.float32).double().reshape(t, k // 32, 2)
        return s["x"][:t * k].view(torch.int8).double().reshape(t, k) * pair[..., 0].repeat_interleave(32, 1)
    if c["x"] == "mxfp8":
        e = s["scales"].int() - 127
        return torch.ldexp(s["x"].view(torch.float8_e4m3fn).double(), e.repeat_interleave(32, 1))
    return s["x"].double()


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "norm":
        h = s["x"].double() + (s["residual"].double() if c["residual"] else 0)
        y = h * torch.rsqrt(h.square().sum(-1, keepdim=True) / c["k"] + EPS) * s["weight"].double()
        h = h if c["residual"] else None
        if c["out"] == "q8":                # nearest code (half away from zero) of each 32 values' largest over 127
            b = y.reshape(c["rows"], -1, 32)
            d = b.abs().amax(-1, keepdim=True) / 127
            q = torch.trunc(b / torch.where(d > 0, d, torch.ones_like(d)) + torch.copysign(torch.full_like(b, 0.5), b))
            return (q * d.half().double()).reshape(y.shape), h
        if c["out"] == "mxfp8":
            a = y.abs().reshape(c["rows"], -1, 32).amax(-1)
            e = torch.where(a > 0, torch.floor(torch.log2(a)) - 7, torch.full_like(a, -127.0)).clamp(-127, 127)
            scaled = y * torch.exp2(-e).repeat_interleave(32, 1)
            step = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp(min=2.0 ** -6))) - 3)
            return (torch.round(scaled / step) * step, torch.exp2(e)), h
        if c["out"] == "f16":
            e = (torch.floor(torch.log2(y.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -200))) - 13).clamp(0, 100)
            return (y * torch.exp2(-e), torch.cat([torch.exp2(-e), torch.exp2(e)], -1)), h
        return y, h
    x = _exact_rows(c, s)
    w = [_exact_weight(PLAIN.get(c["fmt"], c["fmt"]), r) for r in s["raw"]]
    z = [x @ v.T + (b.double() if b is not None else 0) for v, b in zip(w, s["bias"])]
    if c["kind"] == "linear":
        return _act(c["act"], z[0]) + (s["residual"].double() if c["residual"] else 0)
    if c["kind"] == "gate_up":
        return _act(c["act"], z[0]) * z[1]
    gate, dy = z[0].requires_grad_(), s["dy"].double()
    with torch.enable_grad():
        a = _act(c["act"], gate)
    slope = torch.autograd.grad(a, gate, torch.ones_like(a))[0] if a.requires_grad and a is not gate else torch.ones_like(gate)
    dg, du = dy * z[1] * slope, dy * a.detach()
    return dg @ w[0] + du @ w[1], torch.stack([dg, du], 1)
