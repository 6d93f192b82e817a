"""Inputs and 64-bit results of the 4-bit and ragged products' tests, and the bounds their outputs are held to.

Bounds, element by element, from the definition of the kernels' arithmetic (u = 2^-24, a rounding to f32):
  exact products, f32 sums of K terms in any order        K u sum |terms|
  f16 weights f16(s (q - z))                               2^-11 sum |terms| (f16 half a step; below f16's normal range s (q - z) is
                                                           a multiple of the smallest subnormal, as s is, and so exact)
  rows rounded to f16 by row (f32 rows; bf16 rows keep     2^-11 sum |terms| + 2^-38 max |row| sum |w| (a subnormal's half step
  their 8 bits and have the last term alone)               2^-25, the row's largest value being 2^13 or more)
  the output's rounding                                    half a step of its type
"""
import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def w4_raw(g, n, k, group, zeros=True, E=None):
    """(codes, scales, zeros or None, W in 64 bits [E, n, k], its terms' sizes |s| (q + z))."""
    lead = () if E is None else (E,)
    groups = -(-k // group)
    q = torch.randint(0, 16, (*lead, n, k), dtype=torch.uint8, generator=g)
    s = ((torch.rand((*lead, n, groups), generator=g) + 0.5) * 0.02 * torch.where(torch.rand((*lead, n, groups), generator=g) < 0.1, -1, 1)).half()
    z = torch.randint(0, 16, (*lead, n, groups), dtype=torch.uint8, generator=g) if zeros else None
    at = torch.arange(k) // group
    zd = z.double()[..., at] if zeros else 8.0
    w = s.double()[..., at] * (q.double() - zd)
    return q, s, z, w, s.double().abs()[..., at] * (q.double() + zd)


def offsets_of(counts, first=0):
    return torch.tensor([first] + counts).cumsum(0).to(torch.int32)


def spans(offsets, rows):
    """Each expert's (first, end) as the calls read the offsets: clamped, empty where the end is not past the start."""
    o = offsets.clamp(0, rows).tolist()
    return [(a, max(a, b)) for a, b in zip(o[:-1], o[1:])]


def by_expert(x, w, offsets, t=False):
    """x [rows, .] times each expert's w [E, n, k] (transposed product: t) in x's precision; rows of no expert NaN."""
    y = torch.full((x.shape[0], w.shape[2] if t else w.shape[1]), float("nan"), dtype=x.dtype)
    for (a, b), we in zip(spans(offsets, x.shape[0]), w):
        y[a:b] = x[a:b] @ (we if t else we.t())
    return y


def held(got, want, slack, what=""):
    """got against the 64-bit want: off by at most slack and half a step of its type (of the larger of the two)."""
    got = got.detach().cpu()
    g = got.double()
    lim = slack + HALF_STEP[got.dtype] * (want.abs() + slack) + 1e-300
    bad = ~((g - want).abs() <= lim)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, worst {((g - want).abs() / lim).nan_to_num(1e9).max():.3g}"


class Guarded:
    """An output tensor between two sentinel runs: check() says that neither they nor the rows `kept` were written."""
    def __init__(self, shape, dtype, dev, fill=7.25):
        n = 1
        for v in shape:
            n *= v
        self.fill = fill
        self.buf = torch.full((n + 1024,), fill, dtype=dtype, device=dev)
        self.t = self.buf[512:512 + n].view(shape)

    def check(self, kept=()):
        n = self.t.numel()
        assert (self.buf[:512] == self.fill).all() and (self.buf[512 + n:] == self.fill).all(), "written past the output"
        for a, b in kept:
            assert (self.t[a:b] == self.fill).all(), f"rows {a} .. {b - 1} of no expert were written"
