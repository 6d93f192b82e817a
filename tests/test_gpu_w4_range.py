"""Few rows of 4-bit products at the ends of f32's range: a finite answer stays finite though sum x q and sum x of a group are past
the largest f32, and small rows keep their bits.

Bounds as in ragged_case, from the kernels' arithmetic: products exact, f32 sums of K terms |s| |x| (q + z). The sums of a group are
held at 2^-12 of their value, whose smallest step, a subnormal's 2^-149, is 2^-137 of theirs: half of it each time something is added,
2 (k + 8) times an output and sum (the product's, and z times the rows'), times |s| z of at most 16 |s|."""
import pytest
import torch

from qmm import ops
from ragged_case import U, by_expert, gen, held, offsets_of, w4_raw
from test_gpu_w4 import ROW, packed

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16}


def held_scaled(y, want, size, k, s):
    """want, size: in 64 bits; s: the largest scale."""
    tiny = 2 * (k + 8) * 2.0 ** -138 * 16 * s
    assert y.isfinite().all()
    held(y, want, (k + 8) * U * size + tiny)


@pytest.mark.parametrize("rows,n,k,group", [(1, 40, 4096, 128), (1, 24, 160, 32), (2, 17, 512, 64), (5, 33, 2048, ROW), (17, 40, 640, 64), (40, 50, 384, 32),
                                            (20, 4200, 416, 128), (63, 8227, 160, 32), (31, 24, 12288, 128)])
@pytest.mark.parametrize("x_type", ["bf16", "f32"])
@pytest.mark.parametrize("size", [2.0 ** 127, 2.0 ** 118, 2.0 ** -100])
def test_rows_of_any_size(dev, rows, n, k, group, x_type, size):
    g = gen(rows + n)
    q, s, z, w, both = w4_raw(g, n, k, group)
    q, z = torch.randint(12, 16, q.shape, dtype=torch.uint8, generator=g), torch.randint(12, 16, z.shape, dtype=torch.uint8, generator=g)
    s = (s.float() / k).half()   # sums of K values of s (q - z) stay below one
    at = torch.arange(k) // group
    w = s.double()[:, at] * (q.double() - z.double()[:, at])
    both = s.double().abs()[:, at] * (q.double() + z.double()[:, at])
    x = ((torch.rand((rows, k), generator=g) * 0.875 + 1).double() * size).to(T[x_type])   # one sign, below twice the size
    assert x.isfinite().all()
    wp, ws = packed((q, s, z), group, dev)
    y = ops.w4_mm(x.to(dev), wp, ws, n, k, group, out_dtype=torch.float32)
    held_scaled(y, x.double() @ w.t(), x.double() @ both.t(), k, float(s.abs().max()))


@pytest.mark.parametrize("counts", [[1, 0, 3, 2], [1] * 60, [20, 0, 11]])
def test_by_expert(dev, counts):
    rows, E, n, k, g = sum(counts), len(counts), 40, 256, gen(len(counts))
    q, s, z, _, _ = w4_raw(g, n, k, 64, True, E)
    q, z, s = q | 12, z | 12, (s.float() / k).half()
    at = torch.arange(k) // 64
    w = s.double()[..., at] * (q.double() - z.double()[..., at])
    both = s.double().abs()[..., at] * (q.double() + z.double()[..., at])
    wp, ws = packed((q, s, z), 64, dev)
    offsets = offsets_of(counts)
    for x_type in ("bf16", "f32"):
        x = ((torch.rand((rows, k), generator=g) * 0.875 + 1).double() * 2.0 ** 127).to(T[x_type])
        y = ops.w4_mm(x.to(dev), wp, ws, n, k, 64, offsets=offsets.to(dev), out_dtype=torch.float32)
        held_scaled(y, by_expert(x.double(), w, offsets), by_expert(x.double(), both, offsets), k, float(s.abs().max()))


def test_zero_times_large(dev):
    """Codes at their zero point are weights of zero, whatever the row."""
    n, k = 16, 128
    q, s, z = torch.full((n, k), 15, dtype=torch.uint8), torch.full((n, 1), 2.0).half(), torch.full((n, 1), 15, dtype=torch.uint8)
    w, ws = packed((q, s, z), ROW, dev)
    for rows in (1, 5, 40):
        for t in (torch.bfloat16, torch.float32):
            x = torch.full((rows, k), 2.0 ** 127, dtype=t, device=dev)
            assert not ops.w4_mm(x, w, ws, n, k, ROW, out_dtype=torch.float32).any()
