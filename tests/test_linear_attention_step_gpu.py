"""linear_attention_step as a call that writes into a tensor of the user's: what autograd sees of it."""

from __future__ import annotations

import importlib

import pytest
import torch

F = importlib.import_module("hclsm_amd.kernels.linear_attention")


@pytest.fixture
def no_launch(monkeypatch):
    """The call's Python alone, on CPU tensors; yields the argument blocks that would have been launched."""
    blocks = []
    monkeypatch.setattr(F, "require_gpu", lambda *a: None)
    monkeypatch.setattr(F, "_run", lambda name, t, x, *rest: blocks.append(x))
    return blocks


def _token(B=2, H=3, dk=16, dv=24, **kw):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(B, H, d, generator=g).to(**kw) for d in (dk, dk, dv))
    return q, k, v, -torch.rand(H, generator=g).to(**kw), torch.randn(B, H, dk, dv, generator=g).to(**kw)


def test_the_state_counts_as_written(no_launch):
    q, k, v, d, s = _token()
    F.linear_attention_step(q, k, v, d, s)
    assert s._version == 1 and [t._version for t in (q, k, v, d)] == [0] * 4
    pool = torch.zeros(5, 3, 16, 24)
    F.linear_attention_step(q, k, v, d, pool[1:], rows=torch.tensor([0, 3]))
    assert pool._version == 1 and len(no_launch) == 2
    with torch.inference_mode():
        kept = torch.zeros(2, 3, 16, 24)
    with torch.no_grad():
        F.linear_attention_step(q, k, v, d, kept)       # (a state without a version)


@pytest.mark.gpu
def test_a_graph_that_saved_the_state_refuses_its_backward():
    q, k, v, d, s = _token(device="cuda")
    leaf = q[:, None].clone().requires_grad_()
    out = F.linear_attention(leaf, k[:, None], v[:, None], d, initial_state=s)
    (want,) = torch.autograd.grad(out.sum(), leaf, retain_graph=True)
    with torch.no_grad():
        F.linear_attention_step(q, k, v, d, s.clone())
    assert torch.equal(torch.autograd.grad(out.sum(), leaf, retain_graph=True)[0], want)
    with torch.no_grad():
        F.linear_attention_step(q, k, v, d, s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.sum(), leaf)
