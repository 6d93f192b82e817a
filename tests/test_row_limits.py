"""Row counts that no grid holds are refused before a launch (2^24 workgroups of 256 threads are 2^32 threads along x)."""
from test_abi import header_enum, lib  # noqa: F401  (fixture)
from test_sublayer_refusals import F32, at


def test_gate_up_rows(lib):   # noqa: F811
    assert lib.qmm_ffn_gate_up(0, 0, 1 << 24, 32, 8, at(), F32, None, at(), None, at(), None, None, None, at(), F32, None) == header_enum("qmm_status")["QMM_ERR_SHAPE"]
