"""Outputs that share bytes with what they are computed from are refused: other workgroups would read them half written. Exactly the
residual (dh, x of the norm) is taken for an update in place, a neighbour of it is not. Host tensors, nothing is launched."""
import pytest
import torch

from test_sublayer_refusals import ops  # noqa: F401  (fixture)

T, K, N = 4, 512, 512
W = torch.zeros(N * K // 256 * 144, dtype=torch.uint8)


def shifted(rows, cols, by, dtype=torch.float32):
    """Two views [rows, cols] of one buffer, the second by that many elements on."""
    buf = torch.zeros(rows * cols + abs(by), dtype=dtype)
    a, b = buf[:rows * cols].view(rows, cols), buf[abs(by):].view(rows, cols)
    return (a, b) if by >= 0 else (b, a)


@pytest.mark.parametrize("by", [1, K, 3 * K, T * K - 1, -1, -K, 0])
def test_outputs_on_their_inputs(ops, by):   # noqa: F811
    w, one = torch.ones(K), torch.zeros(T, K)
    x, y = shifted(T, K, by)
    calls = [lambda: ops.linear("q4_k", x, W, N, K, y=y, act="silu", q8=False), lambda: ops.ffn_gate_up("q4_k", x, W, W, N, K, y=y, q8=False),
             lambda: ops.gemm_t("q4_k", x, W, N, K, y=y), lambda: ops.rms_norm_backward(x, w, one, dx=y), lambda: ops.rms_norm_backward(one, w, x, dx=y)]
    if by:
        calls += [lambda: ops.linear("q4_k", one, W, N, K, y=y, residual=x, q8=False), lambda: ops.rms_norm(x, w, residual=one, h=y),
                  lambda: ops.rms_norm(one, w, residual=x, h=y), lambda: ops.rms_norm_backward(one, w, one.clone(), dh=x, dx=y)]
    for call in calls:
        with pytest.raises(ValueError, match="overlaps"):
            call()


def test_outputs_on_other_arguments(ops):   # noqa: F811
    big = torch.zeros(1 << 18, dtype=torch.uint8)
    y = big[:T * N * 4].view(torch.float32).view(T, N)
    x, xw, vec = torch.zeros(T, K), big[4096:4096 + W.numel()], big[1024:1024 + 4 * N].view(torch.float32)
    x16, s = torch.zeros(T, K, dtype=torch.float16), big[64:64 + 8 * T].view(torch.float32).view(T, 2)
    res = big[:T * N * 2].view(torch.bfloat16).view(T, N)
    for call in (lambda: ops.linear("q4_k", x, xw, N, K, y=y, q8=False, act="relu"), lambda: ops.linear("q4_k", x, W, N, K, y=y, bias=vec, q8=False),
                 lambda: ops.linear("q4_k", x16, W, N, K, y=y, scales=s), lambda: ops.linear("q4_k", x, W, N, K, y=y, residual=res, q8=False),
                 lambda: ops.ffn_gate_up("q4_k", x, W, xw, N, K, y=y, q8=False), lambda: ops.ffn_gate_up("q4_k", x, W, W, N, K, y=y, bias2=vec, q8=False),
                 lambda: ops.gemm_t("q4_k", x, xw, N, K, y=y),
                 lambda: ops.rms_norm(x, vec, residual=x, h=y), lambda: ops.rms_norm_backward(x, vec, x, dx=y)):
        with pytest.raises(ValueError, match="overlaps"):
            call()


def test_the_tensor_itself_and_its_neighbours_are_taken(ops):   # noqa: F811
    w, one = torch.ones(K), torch.zeros(T, K)
    a, b = shifted(T, K, T * K)   # one after the other
    for call in (lambda: ops.linear("q4_k", one, W, N, K, y=a, residual=a, q8=False), lambda: ops.linear("q4_k", a, W, N, K, y=b, act="silu", q8=False),
                 lambda: ops.ffn_gate_up("q4_k", b, W, W, N, K, y=a, q8=False), lambda: ops.rms_norm(a, w, residual=one, h=a), lambda: ops.rms_norm(one, w, residual=a, h=a),
                 lambda: ops.rms_norm(a, w, residual=a, h=a), lambda: ops.rms_norm(a, w, residual=one, h=b), lambda: ops.rms_norm_backward(one, w, b, dh=a, dx=a)):
        with pytest.raises(AssertionError, match="was reached"):
            call()
