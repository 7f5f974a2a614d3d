"""linear_attention_step as a call that writes into a tensor of the user's: what autograd, transforms and traces see of it, and
its state after thousands of tokens."""

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


@pytest.mark.gpu
@pytest.mark.parametrize("log_decay", [-2.0 ** -12, -1e-6, -3e-5])
def test_thousands_of_tokens(log_decay):
    """float32 states of long memories against float64.  Each token's update rounds the state's element once, by at most
    2^-24 of it, and k v and what is added, which are small beside it; the tokens' values are random, so these roundings are
    independent of each other: after n tokens the rms error is at most sqrt(n) 2^-24 of the largest rms state, and twice that
    with the smaller ones.  (A power of the decay that is itself rounded is off alike for every token: at these decays by 660 to
    1080 times 2^-24 of the state after 4096 tokens.)"""
    n, B, H, dk, dv = 4096, 2, 2, 64, 64
    g = torch.Generator("cuda").manual_seed(4)
    decay = torch.full((H,), log_decay, device="cuda")
    a = torch.exp(decay.double())[:, None, None]
    q, k, v = (torch.randn(n, B, H, d, generator=g, device="cuda") for d in (dk, dk, dv))
    s = 40.0 * torch.randn(B, H, dk, dv, generator=g, device="cuda")
    ref, most = s.double(), 0.0
    for t in range(n):
        F.linear_attention_step(q[t], k[t], v[t], decay, s)
        ref = a * ref + k[t].double()[..., :, None] * v[t].double()[..., None, :]
        if t % 64 == 63:
            most = max(most, ref.square().mean().sqrt().item())
    err = (s.double() - ref).square().mean().sqrt().item()
    assert err <= 2 * n ** 0.5 * 2.0 ** -24 * most, (err / most * 2 ** 24)


def _with_tangents(t):
    return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.gpu
def test_tangents_transforms_and_traces_are_refused():
    """None of these would see what the library does: a call drops tangents, and a trace would hold an empty tensor."""
    from hclsm_amd.kernels import linear_attention_step, residual_rms_norm_fp8
    q, k, v, d, s = _token(device="cuda")
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    before = s.clone()
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        for i in range(5):
            args = [_with_tangents(t) if j == i else t for j, t in enumerate((q, k, v, d, s))]
            with pytest.raises(RuntimeError, match="tangent"):
                linear_attention_step(*args)
        for args in ((_with_tangents(x), x, w), (x, _with_tangents(x), w), (x, x, _with_tangents(w))):
            with pytest.raises(RuntimeError, match="tangent"):
                residual_rms_norm_fp8(*args)
        residual_rms_norm_fp8(x, x, w)      # no input has one
        with pytest.raises(RuntimeError, match="tangent"):
            torch.func.vmap(lambda t: t + residual_rms_norm_fp8(_with_tangents(x))[1].sum())(x)
    with pytest.raises(RuntimeError, match="transform"):
        torch.func.vmap(lambda t: linear_attention_step(t, k, v, d, s))(q[None])
    with pytest.raises(RuntimeError, match="transform"), torch.no_grad():
        torch.func.jvp(lambda t: residual_rms_norm_fp8(t)[1], (x,), (x,))
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda t: linear_attention_step(t, k, v, d, s), (q,))
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda t: residual_rms_norm_fp8(t)[1], (x,))
    assert torch.equal(s, before)


def test_a_state_alone_in_its_pool_may_have_any_stride(no_launch):
    from hclsm_amd import _lib
    q, k, v, d, _ = _token(B=1)
    s = torch.zeros(4, 3 * 16 * 24 + 1)[:, :-1].unflatten(1, (3, 16, 24))[:1]
    assert s.stride(0) % 4 == 1
    F.linear_attention_step(q, k, v, d, s)
    assert _lib.HclsmLinearAttentionStep.from_buffer_copy(no_launch[0]).state_sb == 0


@pytest.mark.gpu
def test_a_state_alone_in_its_pool():
    q, k, v, d, s = _token(B=1, device="cuda")
    odd = torch.zeros(4, 3 * 16 * 24 + 1, device="cuda")[:, :-1].unflatten(1, (3, 16, 24))[:1]
    odd.copy_(s)
    assert torch.equal(F.linear_attention_step(q, k, v, d, odd), F.linear_attention_step(q, k, v, d, s))
    assert torch.equal(odd, s)


def test_a_scalar_is_refused_as_any_other_shape(no_launch):
    q, k, v, d, s = _token()
    with pytest.raises(ValueError, match="q must be"):
        F.linear_attention_step(q[0, 0, 0], k, v, d, s)
    with pytest.raises(ValueError, match="q must be"):
        F.linear_attention(q[0, 0, 0], k, v, d)
