"""What the 4-bit and ragged products refuse, without a device: the C entry points' statuses and the errors of the Python
surface. Nothing is launched."""
import pytest
import torch

from test_abi import header_enum, lib  # noqa: F401  (fixture)
from test_sublayer_refusals import BF16, F16, F32, MXFP8, Q8, at, ops  # noqa: F401  (fixture)

ODD, BYTE = at(0x10008), at(0x10001)


def test_w4_sizes(lib):   # noqa: F811
    assert lib.qmm_w4_bytes(16, 128) == 1024 and lib.qmm_w4_bytes(17, 160) == 4096 and lib.qmm_w4_bytes(1, 32) == 1024
    assert lib.qmm_w4_scale_bytes(17, 160, 64) == 2 * 3 * 64 and lib.qmm_w4_scale_bytes(16, 4096, 1 << 40) == 64
    for n, k in ((0, 32), (8, 0), (8, 33), (-1, 32), ((1 << 20) + 1, 32), (8, (1 << 20) + 32)):
        assert lib.qmm_w4_bytes(n, k) == -1
    for group in (0, 16, 33, 96, -32):
        assert lib.qmm_w4_scale_bytes(8, 256, group) == -1


def test_w4_pack_statuses(lib):   # noqa: F811
    st = header_enum("qmm_status")

    def call(E=1, n=8, k=64, group=32, codes=at(), scales=at(), zeros=None, w=at(), ws=at()):
        return lib.qmm_w4_pack(E, n, k, group, codes, scales, zeros, w, ws, None)

    for bad in (dict(n=0), dict(k=48), dict(k=0), dict(group=48), dict(group=16)):
        assert call(**bad) == st["QMM_ERR_SHAPE"], bad
    for bad in (dict(E=0), dict(E=1025)):
        assert call(**bad) == st["QMM_ERR_RANGE"], bad
    for bad in (dict(codes=None), dict(scales=None), dict(w=None), dict(ws=None)):
        assert call(**bad) == st["QMM_ERR_NULL"], bad
    for bad in (dict(w=ODD), dict(ws=ODD), dict(scales=BYTE)):
        assert call(**bad) == st["QMM_ERR_ALIGN"], bad


def test_w4_mm_statuses(lib):   # noqa: F811
    st = header_enum("qmm_status")

    def mm(rows=4, k=64, n=8, group=32, E=1, off=None, x=at(), xd=BF16, s=None, w=at(), ws=at(), y=at(), yd=F32, work=None, wb=0):
        return lib.qmm_w4_mm(rows, k, n, group, E, off, x, xd, s, w, ws, y, yd, work, wb, None)

    def back(rows=4, k=64, n=8, group=32, E=1, off=None, x=at(), s=at(), w=at(), ws=at(), y=at(), yd=F32, work=None, wb=0):
        return lib.qmm_w4_mm_t(rows, k, n, group, E, off, x, s, w, ws, y, yd, work, wb, None)

    for call in (mm, back):
        for bad in (dict(rows=-1), dict(rows=(1 << 24) + 1), dict(k=40), dict(n=0), dict(group=24), dict(k=(1 << 20) + 32)):
            assert call(**bad) == st["QMM_ERR_SHAPE"], bad
        for bad in (dict(E=0), dict(E=2), dict(E=1025, off=at())):
            assert call(**bad) == st["QMM_ERR_RANGE"], bad
        for bad in (dict(yd=F16), dict(yd=Q8), dict(yd=-1)):
            assert call(**bad) == st["QMM_ERR_DTYPE"], bad
        for bad in (dict(x=None), dict(w=None), dict(ws=None), dict(y=None)):
            assert call(**bad) == st["QMM_ERR_NULL"], bad
        for bad in (dict(x=ODD), dict(w=ODD), dict(ws=ODD), dict(y=at(0x10002)), dict(yd=BF16, y=BYTE), dict(off=at(0x10002)), dict(s=at(0x10002))):
            assert call(**bad) == st["QMM_ERR_ALIGN"], bad
        assert call(rows=0, x=None, w=None, ws=None, y=None) == 0
    assert back(s=None) == st["QMM_ERR_NULL"]
    # few outputs with a long sum: its parts need a workspace
    need = lib.qmm_w4_mm_workspace_size(80, 8192, 64, 1, F16)
    back_need = lib.qmm_w4_mm_t_workspace_size(80, 64, 8192, 1)
    assert need >= 2 * 80 * 64 * 4 and back_need >= 2 * 80 * 64 * 4
    assert lib.qmm_w4_mm_workspace_size(80, 8192, 64, 1, BF16) == 0 and lib.qmm_w4_mm_workspace_size(0, 8192, 64, 1, F16) == 0
    assert lib.qmm_w4_mm_workspace_size(80, 40, 64, 1, F16) == -1 and lib.qmm_w4_mm_t_workspace_size(80, 64, 64, 0) == -1
    for bad in (dict(), dict(work=at(), wb=need - 1), dict(work=None, wb=need)):
        assert mm(rows=80, k=8192, n=64, xd=F16, **bad) == st["QMM_ERR_WORKSPACE"], bad
    assert mm(rows=80, k=8192, n=64, xd=F16, work=ODD, wb=need) == st["QMM_ERR_ALIGN"]
    for bad in (dict(), dict(work=at(), wb=back_need - 1)):
        assert back(rows=80, k=64, n=8192, **bad) == st["QMM_ERR_WORKSPACE"], bad
    assert back(rows=80, k=64, n=8192, work=ODD, wb=back_need) == st["QMM_ERR_ALIGN"]
    for xd in (Q8, MXFP8, -1):
        assert mm(xd=xd) == st["QMM_ERR_DTYPE"]
    # few rows whose row blocks leave CUs without work: K in parts too
    few = lib.qmm_w4_mm_workspace_size(31, 12288, 64, 1, F32)
    assert few >= 2 * 31 * 64 * 4 and lib.qmm_w4_mm_workspace_size(1, 12288, 64, 1, F32) == 0
    for bad in (dict(), dict(work=at(), wb=few - 1)):
        assert mm(rows=31, k=12288, n=64, xd=F32, **bad) == st["QMM_ERR_WORKSPACE"], bad
    assert mm(rows=31, k=12288, n=64, xd=F32, work=ODD, wb=few) == st["QMM_ERR_ALIGN"]


def test_ragged_statuses(lib):   # noqa: F811
    st = header_enum("qmm_status")

    def of(fn):
        return lambda rows=4, k=64, n=8, E=2, off=at(), a=at(), b=at(), d=BF16, y=at(), yd=F32, work=None, wb=0: fn(rows, k, n, E, off, a, b, d, y, yd, work, wb, None)

    for fn in (lib.qmm_ragged_mm, lib.qmm_ragged_mm_t, lib.qmm_ragged_mm_dw):
        call = of(fn)
        for bad in (dict(d=F32), dict(d=Q8), dict(yd=F16), dict(d=F16, yd=BF16)):
            assert call(**bad) == st["QMM_ERR_DTYPE"], bad
        for bad in (dict(rows=-1), dict(rows=(1 << 24) + 1), dict(k=0), dict(k=60), dict(n=12), dict(n=(1 << 20) + 8)):
            assert call(**bad) == st["QMM_ERR_SHAPE"], bad
        for bad in (dict(E=0), dict(E=1025)):
            assert call(**bad) == st["QMM_ERR_RANGE"], bad
        for bad in (dict(off=None), dict(a=None), dict(b=None), dict(y=None)):
            assert call(**bad) == st["QMM_ERR_NULL"], bad
        for bad in (dict(a=ODD), dict(b=ODD), dict(y=ODD), dict(off=at(0x10002))):
            assert call(**bad) == st["QMM_ERR_ALIGN"], bad
    for fn, size, sizes in ((lib.qmm_ragged_mm, lib.qmm_ragged_mm_workspace_size, dict(rows=256, k=65536, n=72, E=1)),
                            (lib.qmm_ragged_mm_t, lib.qmm_ragged_mm_t_workspace_size, dict(rows=80, k=64, n=8192, E=1)),
                            (lib.qmm_ragged_mm_dw, lib.qmm_ragged_mm_dw_workspace_size, dict(rows=8192, k=64, n=64, E=1))):
        need = size(*sizes.values())
        assert need > 0 and size(-1, 64, 64, 1) == -1 and size(80, 60, 64, 1) == -1
        for bad in (dict(), dict(work=at(), wb=need - 1)):
            assert of(fn)(**sizes, **bad) == st["QMM_ERR_WORKSPACE"], bad
        assert of(fn)(**sizes, work=ODD, wb=need) == st["QMM_ERR_ALIGN"]
    assert of(lib.qmm_ragged_mm)(rows=0, a=None, y=None) == 0
    assert of(lib.qmm_ragged_mm_t)(rows=0, a=None, y=None) == 0


def w4(n=8, k=64, group=32, E=1):
    blocks, tiles, groups = -(-n // 16), -(-k // 128), -(-k // group)
    return torch.zeros(E * blocks * tiles * 1024, dtype=torch.uint8), torch.zeros(E * blocks * groups * 16, dtype=torch.int32)


def test_w4_surface(ops):   # noqa: F811
    w, ws = w4()
    x, dy, off = torch.zeros(4, 64), torch.zeros(4, 8), torch.zeros(2, dtype=torch.int32)
    half = torch.zeros(4, 64, dtype=torch.float16)
    wrong = [
        lambda: ops.w4_pack(torch.zeros(8, 64), torch.zeros(8, 2).half(), group=32),
        lambda: ops.w4_pack(torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(8, 2), group=32),
        lambda: ops.w4_pack(torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(8, 1).half(), group=32),
        lambda: ops.w4_pack(torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(8, 2).half(), torch.zeros(8, 2), group=32),
        lambda: ops.w4_pack(torch.zeros(8, 48, dtype=torch.uint8), torch.zeros(8, 2).half(), group=32),
        lambda: ops.w4_pack(torch.zeros(64, dtype=torch.uint8), torch.zeros(2).half(), group=32),
        lambda: ops.w4_mm(x, w[:-1], ws, 8, 64, 32), lambda: ops.w4_mm(x, w, ws[:-1], 8, 64, 32), lambda: ops.w4_mm(x, w, ws, 8, 64, 64),
        lambda: ops.w4_mm(x, w, ws, 8, 64, 48), lambda: ops.w4_mm(x, w, ws, 24, 64, 32), lambda: ops.w4_mm(x[:, :32].contiguous(), w, ws, 8, 64, 32),
        lambda: ops.w4_mm(x[0], w, ws, 8, 64, 32), lambda: ops.w4_mm(x[:, ::2], w, ws, 8, 32, 32), lambda: ops.w4_mm(x.double(), w, ws, 8, 64, 32),
        lambda: ops.w4_mm(x, w, ws, 8, 64, 32, scales=torch.ones(4, 2)), lambda: ops.w4_mm(half, w, ws, 8, 64, 32, scales=torch.ones(3, 2)),
        lambda: ops.w4_mm(x, w, ws, 8, 64, 32, offsets=off.long()), lambda: ops.w4_mm(x, w, ws, 8, 64, 32, offsets=off[:1]),
        lambda: ops.w4_mm(x, w, ws, 8, 64, 32, offsets=torch.zeros(3, dtype=torch.int32)),
        lambda: ops.w4_mm(x, w, ws, 8, 64, 32, y=torch.zeros(4, 9)), lambda: ops.w4_mm(x, w, ws, 8, 64, 32, out_dtype=torch.float16),
        lambda: ops.w4_mm(x, w, ws, 8, 64, 32, y=x.view(-1)[8:40].view(4, 8)), lambda: ops.w4_mm(x, w, ws, 8, 64, 32, y=w.view(torch.float32)[:32].view(4, 8)),
        lambda: ops.w4_mm_t(dy[:, :4].contiguous(), w, ws, 8, 64, 32), lambda: ops.w4_mm_t(dy.half(), w, ws, 8, 64, 32),
        lambda: ops.w4_mm_t(dy[0], w, ws, 8, 64, 32), lambda: ops.w4_mm_t(dy, w, ws[1:], 8, 64, 32),
        lambda: ops.w4_mm_t(dy, w, ws, 8, 64, 32, y=w.view(torch.float32).view(4, 64)),
    ]
    for i, call in enumerate(wrong):
        with pytest.raises(ValueError):
            print("call", i)
            call()


def test_ragged_surface(ops):   # noqa: F811
    x, dy, w = torch.zeros(4, 64).bfloat16(), torch.zeros(4, 16).bfloat16(), torch.zeros(2, 16, 64).bfloat16()
    off = torch.zeros(3, dtype=torch.int32)
    wrong = [
        lambda: ops.ragged_mm(x, off[:2], w), lambda: ops.ragged_mm(x, off.long(), w), lambda: ops.ragged_mm(x, off, w[0]),
        lambda: ops.ragged_mm(x.float(), off, w), lambda: ops.ragged_mm(x.half(), off, w), lambda: ops.ragged_mm(x, off, w.float()),
        lambda: ops.ragged_mm(x[:, :32].contiguous(), off, w), lambda: ops.ragged_mm(x[0], off, w), lambda: ops.ragged_mm(x, off, w.transpose(1, 2)),
        lambda: ops.ragged_mm(x, off, w, out_dtype=torch.float16), lambda: ops.ragged_mm(x, off, w, y=torch.zeros(4, 8)),
        lambda: ops.ragged_mm(x, off, w, y=torch.zeros(4, 16), out_dtype=torch.bfloat16), lambda: ops.ragged_mm(x, off, w, y=x.view(-1)[:64].view(4, 16)),
        lambda: ops.ragged_mm_t(dy[:, :8].contiguous(), off, w), lambda: ops.ragged_mm_t(dy.half(), off, w), lambda: ops.ragged_mm_t(dy, off, w, dx=w[0, :4]),
        lambda: ops.ragged_mm_t(dy[0], off, w), lambda: ops.ragged_mm_dw(dy[:3], x, off), lambda: ops.ragged_mm_dw(dy.half(), x, off),
        lambda: ops.ragged_mm_dw(dy.float(), x.float(), off), lambda: ops.ragged_mm_dw(dy[0], x, off), lambda: ops.ragged_mm_dw(dy, x, off, dw=torch.zeros(2, 64, 16)),
        lambda: ops.ragged_mm_dw(dy, x, off.float()),
        lambda: ops.ragged_mm_backward(dy[:3], x, off, w), lambda: ops.ragged_mm_backward(dy, x[:3], off, w), lambda: ops.ragged_mm_backward(dy.half(), x, off, w),
        lambda: ops.ragged_mm_backward(dy, x.half(), off, w), lambda: ops.ragged_mm_backward(dy, dy, off, w), lambda: ops.ragged_mm_backward(dy, x, off, w.float()),
        lambda: ops.ragged_mm_backward(dy, x, off[:2], w), lambda: ops.ragged_mm_backward(dy, x, off, w, out_dtype=torch.float16),
        lambda: ops.ragged_mm_backward(dy, x, off, w, dw_dtype=torch.float16), lambda: ops.ragged_mm_backward(dy[0], x, off, w),
    ]
    for i, call in enumerate(wrong):
        with pytest.raises(ValueError):
            print("call", i)
            call()


def test_good_calls_reach_the_library(ops):   # noqa: F811
    w, ws = w4()
    x = torch.zeros(4, 64)
    off = torch.zeros(3, dtype=torch.int32)
    w2, ws2 = w4(E=2)
    r = torch.zeros(2, 16, 64).bfloat16()
    for call in (lambda: ops.w4_mm(x, w, ws, 8, 64, 32), lambda: ops.w4_mm(x.half(), w, ws, 8, 64, 32, y=torch.zeros(4, 8)),
                 lambda: ops.w4_mm(x, w2, ws2, 8, 64, 32, offsets=off), lambda: ops.w4_mm_t(torch.zeros(4, 8), w, ws, 8, 64, 32),
                 lambda: ops.ragged_mm(x.bfloat16(), off, r), lambda: ops.ragged_mm_t(torch.zeros(4, 16).bfloat16(), off, r),
                 lambda: ops.ragged_mm_dw(torch.zeros(4, 16).bfloat16(), x.bfloat16(), off)):
        with pytest.raises(AssertionError, match="was reached"):
            call()


def test_w4_scale_words_past_31_bits(lib, ops):   # noqa: F811
    """2^20 rows of 16384 values in groups of 32: 2^31 bytes of scale words."""
    n, k, group = 1 << 20, 16384, 32
    assert lib.qmm_w4_scale_bytes(n, k, group) == 1 << 31 and lib.qmm_w4_bytes(n, k) == 1 << 33
    assert lib.qmm_w4_scale_bytes(1 << 20, 1 << 20, 32) == 1 << 37 and lib.qmm_w4_scale_bytes((1 << 20) + 1, k, group) == -1
    assert ops._w4_sizes(n, k, group) == (1 << 33, 1 << 31)
    st = header_enum("qmm_status")
    assert lib.qmm_w4_pack(1, n, k, group, None, None, None, None, None, None) == st["QMM_ERR_NULL"]


def test_rows_of_no_expert_flag(lib):   # noqa: F811
    """QMM_ZERO_REST comes with the types that a call takes; the weights' gradient has no such rows."""
    import re
    from test_abi import HEADER
    from qmm import ops
    rest = int(re.search(r"#define QMM_ZERO_REST (\d+)", open(HEADER).read()).group(1))
    st = header_enum("qmm_status")
    assert ops._ZERO_REST == rest
    for yd, good in ((F32, True), (BF16, True), (F16, False), (Q8, False), (-1, False), (2 * rest, False)):
        want = 0 if good else st["QMM_ERR_DTYPE"]
        assert lib.qmm_w4_mm(0, 64, 8, 32, 2, at(), None, BF16, None, None, None, None, yd | rest, None, 0, None) == want
        assert lib.qmm_w4_mm_t(0, 64, 8, 32, 2, at(), None, None, None, None, None, yd | rest, None, 0, None) == want
        for fn in (lib.qmm_ragged_mm, lib.qmm_ragged_mm_t):
            assert fn(0, 64, 8, 2, at(), None, at(), BF16, None, yd | rest, None, 0, None) == want
    assert lib.qmm_w4_mm(0, 64, 8, 32, 1, None, None, BF16, None, None, None, None, F32 | rest, None, 0, None) == 0
    assert lib.qmm_ragged_mm_dw(4, 64, 8, 2, at(), at(), at(), BF16, at(), F32 | rest, None, 0, None) == st["QMM_ERR_DTYPE"]


def test_ragged_products_need_offsets(ops):   # noqa: F811
    """None means one matrix for all rows to the 4-bit products alone."""
    x, dy, w = torch.zeros(4, 64).bfloat16(), torch.zeros(4, 16).bfloat16(), torch.zeros(1, 16, 64).bfloat16()
    for call in (lambda: ops.ragged_mm(x, None, w), lambda: ops.ragged_mm_t(dy, None, w), lambda: ops.ragged_mm_dw(dy, x, None),
                 lambda: ops.ragged_mm_backward(dy, x, None, w)):
        with pytest.raises(ValueError, match="offsets"):
            call()


def test_exact_products_take_no_operand(ops):   # noqa: F811
    w, ws = w4()
    with pytest.raises(ValueError, match="exact"):
        ops.w4_mm(torch.zeros(80, 64).half(), w, ws, 8, 64, 32, exact=True)
