"""Formats that the products with an epilogue do not take are ValueErrors that name the format: a gate / up pair in two formats (the
plain swiglu's "gate+up"), and names that are no format. Host tensors, nothing is launched."""
import pytest
import torch

from test_sublayer_refusals import ops  # noqa: F401  (fixture)


@pytest.mark.parametrize("fmt", ["q4_k+q6_k", "q4_k+q4_k", "q5_k", None])
def test_formats(ops, fmt):   # noqa: F811
    n, k = 32, 512
    w, x, b, dy = torch.zeros(n * k // 256 * 210, dtype=torch.uint8), torch.zeros(2, k), torch.zeros(n), torch.zeros(2, n)
    for call in (lambda: ops.linear(fmt, x, w, n, k, bias=b), lambda: ops.ffn_gate_up(fmt, x, w, w, n, k), lambda: ops.gemm_t(fmt, dy, w, n, k),
                 lambda: ops.linear_backward(fmt, x, w, dy, n, k), lambda: ops.ffn_gate_up_backward(fmt, x, w, w, dy, n, k)):
        with pytest.raises(ValueError, match=(fmt or "None").replace("+", r"\+")):
            call()
