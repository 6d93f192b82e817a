"""The measured calls of 4-bit weights with group scales and of products grouped by expert with ragged sizes, through
``qmm.ops``.

    w4_mm             y = x W^T, W[r, c] = s[r, c / group] (q[r, c] - z[r, c / group]) with 4-bit codes q, f16 scales and
                      4-bit zero points; dense, or by expert: rows offsets[e] .. offsets[e + 1] - 1 times expert e's matrix
    w4_mm_t           dx = dy W, the input gradient through those weights (frozen)
    ragged_mm         y = x W_e^T over 16-bit expert weights, rows sorted by expert
    ragged_mm_backward  its gradients dx = dy W_e and dW_e = dy_e^T x_e

The listed cases are these calls at the sizes of this repository's dense layers (hidden 4096, FFN 12288) and expert layers
(2048 / 768 with 128 experts and 8 a token, 2880 with 32 experts and 4 a token), from one decoded token to prompts and
training batches of thousands; ``draw`` takes any type, group, number of experts and size of the same ranges.

Weights are quantized from values of a trained layer's size; activations are rows of unit variance; experts are hit as a
router hits them, some often and some not at all. ``own`` False computes the plain form in 32 bits.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _ops():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "loom-skills_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from qmm import ops
    return ops


def _w4(name, kind, rows, n, k, group, zeros, x="bf16", out="bf16", experts=0):
    return {"name": name, "kind": kind, "rows": rows, "n": n, "k": k, "group": group, "zeros": zeros, "x": x, "out": out,
            "experts": experts}


def _ragged(name, kind, rows, n, k, experts, x="bf16", out="bf16"):
    return {"name": name, "kind": kind, "rows": rows, "n": n, "k": k, "x": x, "out": out, "experts": experts}


def listed():
    return [
        # a projection of one decoded token: a decode step's weight stream
        _w4("w4 mv 1 token 12288 x 4096", "w4", 1, 12288, 4096, 128, True, "bf16", "bf16"),
        # a few drafted tokens on f32 rows
        _w4("w4 mv 5 tokens 6144 x 2048", "w4", 5, 6144, 2048, 32, True, "f32", "f32"),
        # a ragged prompt chunk
        _w4("w4 gemm 333 rows 12288 x 4096", "w4", 333, 12288, 4096, 128, True),
        # a long prompt through the down projection, symmetric codes
        _w4("w4 gemm 2048 rows 4096 x 12288", "w4", 2048, 4096, 12288, 64, False),
        # gate and up (one tensor) of 13 decoded tokens' experts: fewer rows than experts
        _w4("w4 experts 104 rows 1536 x 2048", "w4", 104, 1536, 2048, 128, True, "bf16", "f32", 128),
        # the same experts for a prompt of 1000 tokens
        _w4("w4 experts 8000 rows 1536 x 2048", "w4", 8000, 1536, 2048, 128, True, "bf16", "bf16", 128),
        # the input gradient of a small layer for a short batch
        _w4("w4 grad 77 rows 768 x 2048", "w4_t", 77, 768, 2048, 32, True),
        # the input gradient of a dense layer's projection for a training batch
        _w4("w4 grad 2048 rows 12288 x 4096", "w4_t", 2048, 12288, 4096, 128, True),
        # one decoded token through its four experts' up projection
        _ragged("experts 4 rows 2880 x 2880", "ragged", 4, 2880, 2880, 32),
        # a training batch through fine-grained experts' up projection: gradients of the input and of the weights
        _ragged("experts grad 8000 rows 768 x 2048", "ragged_grad", 8000, 768, 2048, 128, "bf16", "f32"),
        # a long batch through coarse experts, forward and then both gradients
        _ragged("experts 16384 rows 2880 x 2880", "ragged", 16384, 2880, 2880, 32),
        _ragged("experts grad 16384 rows 2880 x 2880", "ragged_grad", 16384, 2880, 2880, 32, "bf16", "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["w4", "w4", "w4", "w4_t", "ragged", "ragged", "ragged_grad", "ragged_grad"])
    if kind in ("w4", "w4_t"):
        experts = rng.choice([0, 0, _log_int(rng, 2, 128)])
        k = 32 * _log_int(rng, 8, 384)
        n = _log_int(rng, 64, 12288)
        if experts:
            n, k = min(n, 4096), min(k, 4096)
            experts = max(1, min(experts, int(5e8 / (n * k))))
        few = kind == "w4" and rng.random() < 0.5
        rows = _log_int(rng, 1, 32) if few else _log_int(rng, 64, 8192)
        rows = max(1, min(rows, int(4e11 / (2 * n * k))))
        few = few or rows < 64
        x = rng.choice(["bf16", "f32"]) if few and kind == "w4" else "bf16"
        out = rng.choice(["bf16", "f32"]) if few and kind == "w4" else "bf16"
        c = _w4("", kind, rows, n, k, rng.choice([32, 64, 128, 256, 1 << 20]), rng.random() < 0.6, x, out, experts)
    else:
        experts = _log_int(rng, 1, 160)
        n, k = 8 * _log_int(rng, 8, 720), 8 * _log_int(rng, 8, 720)
        experts = max(1, min(experts, int(2e8 / (n * k))))
        rows = _log_int(rng, 1, 16384)
        rows = max(1, min(rows, int((5e11 if kind == "ragged" else 2.5e11) / (2 * n * k))))
        x = rng.choice(["bf16", "bf16", "f16"])
        c = _ragged("", kind, rows, n, k, experts, x, rng.choice([x, "f32"]))
    del c["name"]
    return c


# -------------------------------------------------------------------------------------------------------- inputs
def _quantized(g, n, k, group, zeros):
    """(codes u8 [n, k], scales f16 [n, groups], zero points u8 [n, groups]) of normal weights of about 1 / sqrt(k), by the
    smallest and largest value of a group, or symmetric about code 8."""
    w = torch.randn((n, k), device=DEV, generator=g) / math.sqrt(k)
    groups = -(-k // group)
    size = min(group, k)
    v = torch.nn.functional.pad(w, (0, groups * size - k)).reshape(n, groups, size)
    if zeros:
        lo, hi = v.amin(-1).clamp(max=0), v.amax(-1).clamp(min=0)
        s = ((hi - lo) / 15).half()
        z = torch.round(-lo / s.float()).clamp(0, 15)
    else:
        s = (v.abs().amax(-1) / 7.5).half()
        z = torch.full_like(s, 8, dtype=torch.float32)
    q = torch.round(v / s.float()[..., None] + z[..., None]).clamp(0, 15).to(torch.uint8)
    return q.reshape(n, -1)[:, :k].contiguous(), s, z.to(torch.uint8)


def _stored(q, s, z):
    """The weights as a program keeps them (what ops.w4_pack lays out once): tiles of 16 rows x 128 values, 1 KB each, lane
    16 h + r holding values 32 j + 8 h .. + 7 of row r in its word j, values 0-3 of the eight in the low nibbles; and a word
    (f16 scale, f16 1024 + zero point) a row and group, [rows / 16][groups][16]."""
    n, k = q.shape
    np_, kp = -(-n // 16) * 16, -(-k // 128) * 128
    t = torch.nn.functional.pad(q, (0, kp - k, 0, np_ - n))
    t = t.reshape(np_ // 16, 16, kp // 128, 4, 4, 2, 4)         # row, tile, j, h, half, byte
    t = (t[..., 0, :] | (t[..., 1, :] << 4)).permute(0, 2, 4, 1, 3, 5)
    words = s.view(torch.int16).int() & 0xFFFF | (z.int() | 0x6400) << 16
    words = torch.nn.functional.pad(words, (0, 0, 0, np_ - n), value=0x64000000)
    return t.reshape(-1).contiguous(), words.reshape(np_ // 16, 16, -1).permute(0, 2, 1).contiguous().reshape(-1)


def _counts(rows, experts, seed):
    """Rows of each expert, as a router deals them: uneven, some experts without any."""
    g = torch.Generator()
    g.manual_seed(seed)
    p = torch.exp(0.8 * torch.randn(experts, generator=g)) * (torch.rand(experts, generator=g) > 0.08)
    p = p + 1e-9
    return torch.bincount(torch.multinomial(p, rows, replacement=True, generator=g), minlength=experts).tolist()


def prepare(case, seed):
    c, g = case, torch.Generator(device=DEV)
    g.manual_seed(seed)
    n, k, rows, experts = c["n"], c["k"], c["rows"], c["experts"]
    s = {"c": c, "offsets": None, "spans": [(0, rows)]}
    if experts:
        ends = torch.tensor([0] + _counts(rows, experts, seed + 1)).cumsum(0)
        s["offsets"] = ends.to(torch.int32).to(DEV)
        s["spans"] = list(zip(ends[:-1].tolist(), ends[1:].tolist()))
    if c["kind"] in ("w4", "w4_t"):
        s["raw"] = [_quantized(g, n, k, c["group"], c["zeros"]) for _ in range(max(1, experts))]
        packed = [_stored(*r) for r in s["raw"]]
        s["w"], s["ws"] = torch.cat([p[0] for p in packed]), torch.cat([p[1] for p in packed])
    else:
        s["w"] = torch.empty((experts, n, k), dtype=TYPE[c["x"]], device=DEV)
        s["w"].normal_(0, 1 / math.sqrt(k), generator=g)
    if c["kind"] != "w4_t":
        s["x"] = torch.randn((rows, k), device=DEV, generator=g).to(TYPE[c["x"]])
    if c["kind"] in ("w4_t", "ragged_grad"):
        s["dy"] = (1e-2 * torch.randn((rows, n), device=DEV, generator=g)).to(TYPE[c["x"]])
    return s


# ----------------------------------------------------------------------------------------------- the plain form
def _values(raw, group):
    """W in 32 bits [n, k]."""
    q, s, z = raw
    at = torch.arange(q.shape[1], device=DEV) // group
    return s.float()[:, at] * (q.float() - z.float()[:, at])


def _plain(s):
    c = s["c"]
    out = TYPE[c["out"]]
    if c["kind"] == "w4":
        x = s["x"].float()
        return torch.cat([torch.matmul(x[a:b], _values(r, c["group"]).t()) for (a, b), r in zip(s["spans"], s["raw"]) if a < b]).to(out)
    if c["kind"] == "w4_t":
        dy = s["dy"].float()
        return torch.cat([torch.matmul(dy[a:b], _values(r, c["group"])) for (a, b), r in zip(s["spans"], s["raw"]) if a < b]).to(out)
    x = s["x"].float()
    parts = [(a, b, w) for (a, b), w in zip(s["spans"], s["w"])]
    if c["kind"] == "ragged":
        return torch.cat([torch.matmul(x[a:b], w.float().t()) for a, b, w in parts if a < b]).to(out)
    dy = s["dy"].float()
    dx = torch.cat([torch.matmul(dy[a:b], w.float()) for a, b, w in parts if a < b]).to(out)
    return dx, torch.stack([torch.matmul(dy[a:b].t(), x[a:b]).to(out) for a, b, _ in parts])


def run(state):
    s, c = state, state["c"]
    if not own:
        return _plain(s)
    ops = _ops()
    out = TYPE[c["out"]]
    if c["kind"] == "w4":
        return ops.w4_mm(s["x"], s["w"], s["ws"], c["n"], c["k"], c["group"], offsets=s["offsets"], out_dtype=out)
    if c["kind"] == "w4_t":
        return ops.w4_mm_t(s["dy"], s["w"], s["ws"], c["n"], c["k"], c["group"], offsets=s["offsets"], out_dtype=out)
    if c["kind"] == "ragged":
        return ops.ragged_mm(s["x"], s["offsets"], s["w"], out_dtype=out)
    return ops.ragged_mm_backward(s["dy"], s["x"], s["offsets"], s["w"], out_dtype=out, dw_dtype=out)


# -------------------------------------------------------------------------------------------------------- work
def _size(t):
    return 4 if t == "f32" else 2


def work(case):
    c = case
    n, k, rows, e = c["n"], c["k"], c["rows"], max(1, c["experts"])
    hit = e if c["experts"] == 0 else _hit(rows, e)
    if c["kind"] in ("w4", "w4_t"):
        weights = hit * n * (k // 2 + 4 * -(-k // c["group"]))
        wide, narrow = (k, n) if c["kind"] == "w4" else (n, k)
        return {"bytes": weights + rows * (wide * _size(c["x"]) + narrow * _size(c["out"])), "flops": 2 * rows * n * k}
    if c["kind"] == "ragged":
        return {"bytes": 2 * hit * n * k + rows * (2 * k + n * _size(c["out"])), "flops": 2 * rows * n * k}
    size = _size(c["out"])
    return {"bytes": 2 * hit * n * k + e * n * k * size + rows * (2 * k + 2 * n + k * size), "flops": 4 * rows * n * k}


def _hit(rows, experts):
    """About how many of the experts have a row at all."""
    return max(1, min(experts, round(0.92 * experts * (1 - math.exp(-0.8 * rows / experts)))))


# ----------------------------------------------------------------------------------------- the results in 64 bits
def _exact_weight(raw, group):
    """W in 64 bits from its definition, a group at a time."""
    q, s, z = raw[0], raw[1].double(), raw[2].double()
    parts = q.double().split(group, 1)
    return torch.cat([(p - z[:, i:i + 1]) * s[:, i:i + 1] for i, p in enumerate(parts)], 1)


def exact(case, seed):
    c = case
    if c["rows"] * c["n"] * c["k"] > 1.5e11:
        return None
    s = prepare(c, seed)
    four_bit = c["kind"] in ("w4", "w4_t")
    back = c["kind"] in ("w4_t", "ragged_grad")
    y = torch.empty((c["rows"], c["k"] if back else c["n"]), dtype=torch.float64, device=DEV)
    dw = None if c["kind"] != "ragged_grad" else torch.zeros((c["experts"], c["n"], c["k"]), dtype=torch.float64, device=DEV)
    for e, (a, b) in enumerate(s["spans"]):
        if a == b:
            continue
        w = _exact_weight(s["raw"][e], c["group"]) if four_bit else s["w"][e].double()
        if not back:
            y[a:b] = (w @ s["x"][a:b].double().t()).t()
            continue
        y[a:b] = (w.t() @ s["dy"][a:b].double().t()).t()
        if dw is not None:
            dw[e] = (s["x"][a:b].double().t() @ s["dy"][a:b].double()).t()
    return y if dw is None else (y, dw)
