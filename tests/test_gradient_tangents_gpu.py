"""A gradient with a tangent (forward mode over reverse) is refused by the operators whose backward runs in the library: it would be
dropped there without a word."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def _calls():
    from hclsm_amd.kernels import RotaryPlan, cross_attention, linear_attention, qk_norm_rotary, residual_rms_norm, rotary_embedding
    x = torch.randn(2, 8, 3, 16, device="cuda")
    d, plan = torch.zeros(3, device="cuda"), RotaryPlan(16)
    return x, {"linear_attention": lambda t: linear_attention(t, x, x, d), "residual_rms_norm": lambda t: residual_rms_norm(t, x)[0],
               "cross_attention": lambda t: cross_attention(t, x, x), "rotary_embedding": lambda t: rotary_embedding(t, plan),
               "qk_norm_rotary": lambda t: qk_norm_rotary(t, x, torch.ones(16, device="cuda"), torch.ones(16, device="cuda"), plan)[0]}


@pytest.mark.parametrize("name", ["linear_attention", "residual_rms_norm", "cross_attention", "rotary_embedding", "qk_norm_rotary"])
def test_a_tangent_of_a_gradient_is_refused(name):
    x, calls = _calls()
    t = x.clone().requires_grad_()
    out = calls[name](t)
    g = torch.randn_like(out)
    (want,) = torch.autograd.grad(out, t, g, retain_graph=True)
    with forward_ad.dual_level():
        assert torch.equal(torch.autograd.grad(out, t, g, retain_graph=True)[0], want)      # no tangent: as ever
        with pytest.raises(RuntimeError, match="tangent"):
            torch.autograd.grad(out, t, forward_ad.make_dual(g, torch.ones_like(g)))
