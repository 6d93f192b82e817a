"""The feed-forward examples of INTEGRATION.md, run as they stand: the inference block against the 64-bit sub-layer, the training
block's gradients against autograd in 64 bits, its inputs unchanged."""
import os
import re

import numpy as np
import pytest
import torch

from helpers import assert_close_rel_l2
from sublayer import U8, Weight, f64, glu64, rows, vec

pytestmark = pytest.mark.gpu
EPS = 1e-6
DOC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")


def _block(word):
    blocks = [b for b in re.findall(r"^```python\n(.*?)^```", open(DOC).read(), flags=re.S | re.M) if word in b]
    assert len(blocks) == 1, f"{len(blocks)} examples with {word}"
    return blocks[0]


def _names(dev, T):
    from qmm import ops
    rng = np.random.default_rng(T)
    H, F = 512, 1024
    w = {"w_gate": Weight("q4_k", rng, F, H, dev), "w_up": Weight("q4_k", rng, F, H, dev), "w_down": Weight("q6_k", rng, H, F, dev)}
    d = {"attn_out": rows(rng, (T, H), torch.bfloat16, dev), "h": rows(rng, (T, H), torch.bfloat16, dev), "dy": rows(rng, (T, H), torch.bfloat16, dev, 1e-3),
         "norm_w": 1 + vec(rng, H, dev, 0.1)}
    return w, d, dict(d, **{n: v.w for n, v in w.items()}, ops=ops, torch=torch, eps=EPS, H=H, F=F, T=T)


def _normed(h, w):
    return h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS) * w


def test_inference(dev):
    """rel-L2 2e-2: two Q8_1 operands, each off by at most half a step of 2^-7 of its 32 values' largest."""
    w, d, names = _names(dev, 5)
    h = f64(d["attn_out"]) + f64(d["h"])
    W = {n: torch.from_numpy(v.W) for n, v in w.items()}
    y = _normed(h, f64(d["norm_w"]))
    want = h + glu64("silu", y @ W["w_gate"].T, y @ W["w_up"].T) @ W["w_down"].T
    exec(_block("residual=h, y=h"), names)
    assert names["h"] is d["h"]
    assert_close_rel_l2(f64(names["h"]).numpy(), want.numpy(), 2e-2, "h")


@pytest.mark.parametrize("T", [70, 200])
def test_training(dev, T):
    """da, dgu and dn are bf16 rows: 1.7e-3 rms each (half a step of 2^-8 over sqrt 3, and over the binade), 3e-3 together with the
    f16 operands; three times that. dh is rounded once more."""
    w, d, names = _names(dev, T)
    before = {n: t.clone() for n, t in d.items()}
    exec(_block("rms_norm_backward("), names)
    assert all(torch.equal(d[n], before[n]) for n in d)
    h, nw = (f64(d["attn_out"]) + f64(d["h"])).requires_grad_(), f64(d["norm_w"]).requires_grad_()
    y = _normed(h, nw)
    y = y + (f64(names["x16"]) * f64(names["s"][:, 1:]) - y).detach()   # at the operand that the kernels multiply
    W = {n: torch.from_numpy(v.W16) for n, v in w.items()}
    part = glu64("silu", y @ W["w_gate"].T, y @ W["w_up"].T) @ W["w_down"].T
    part.backward(f64(d["dy"]))
    got = f64(names["dh"])
    assert (got - f64(d["dy"]) - h.grad).norm() <= 1e-2 * h.grad.norm() + U8 * got.norm()
    assert_close_rel_l2(f64(names["dw"]).numpy(), nw.grad.numpy(), 1e-2, "dw")
    assert_close_rel_l2(f64(names["y"]).numpy(), (h + part).detach().numpy(), 1e-2, "y")
