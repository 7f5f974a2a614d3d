"""Linear attention and norms with the residual together, as one layer of a residual stream uses them: a training step with
gradients through two layers against float64 autograd, and a prompt with single tokens behind it against the whole sequence.

    y, h = residual_rms_norm(x, h, w);  q, k, v = y W;  x = linear_attention(q, k, v) W_o;  next layer

Tolerances are by norm: every tensor between two float32 operators is off by at most the sum of their own errors, each below
2e-6 of its norm (test_linear_attention_gpu.py, test_residual_norm_gpu.py; products of 96 terms: 96 * 2^-24 = 6e-6 at most),
through 12 operators forward and as many back: 24 * 6e-6 < 2e-4 of the largest intermediate gradient, which is within a factor of
ten of the results here.  bf16 tensors are off by half a step, 2^-8, each, through 8 roundings in a row: 2^-5."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

H, HK, DK, DV, D = 6, 2, 16, 24, 96


def _weights(g, layers=2):
    mk = lambda *s: torch.randn(*s, generator=g) / s[0] ** 0.5
    return [dict(w=1 + 0.1 * torch.randn(D, generator=g), qkv=mk(D, H * DK + HK * (DK + DV)), o=mk(H * DV, D)) for _ in range(layers)]


def _split(p, B, L):
    q, k, v = p.split((H * DK, HK * DK, HK * DV), -1)
    return q.reshape(B, L, H, DK), k.reshape(B, L, HK, DK), v.reshape(B, L, HK, DV)


def _run(x, layers, decay, states=None):
    from hclsm_amd.kernels import linear_attention, residual_rms_norm
    B, L, _ = x.shape
    h, new = torch.zeros_like(x), []
    for i, p in enumerate(layers):
        y, h = residual_rms_norm(x, h, p["w"])
        out, s = linear_attention(*_split(y @ p["qkv"], B, L), decay, initial_state=None if states is None else states[i],
                                  return_state=True)
        new.append(s)
        x = out.reshape(B, L, H * DV) @ p["o"]
    y, h = residual_rms_norm(x, h)
    return y, new


def _plain(x, layers, decay):
    """The same in elementary float64 operations."""
    B, L, _ = x.shape
    h = torch.zeros_like(x)
    norm = lambda t, w: t / (t.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w
    age = torch.arange(L, device=x.device)[:, None] - torch.arange(L, device=x.device)[None]
    w = torch.where(age >= 0, torch.exp(decay.double()[:, None, None] * age.clamp(min=0)), 0.0)
    for p in layers:
        h = x + h
        q, k, v = _split(norm(h, p["w"]) @ p["qkv"], B, L)
        k, v = (t.repeat_interleave(H // HK, 2).transpose(1, 2) for t in (k, v))
        pairs = torch.matmul(q.transpose(1, 2), k.transpose(-1, -2).contiguous()) * DK ** -0.5 * w
        x = torch.matmul(pairs, v).transpose(1, 2).reshape(B, L, H * DV) @ p["o"]
    return norm(x + h, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_step(dtype):
    g = torch.Generator().manual_seed(1)
    x, gy = torch.randn(3, 150, D, generator=g), torch.randn(3, 150, D, generator=g)
    layers = _weights(g)
    decay = -torch.tensor([0.0, 0.01, 0.1, 0.5, 0.002, 3.0]).cuda()
    cast = lambda t, dt: t.to(dtype).cuda().to(dt).requires_grad_()
    for dt, fn in ((dtype, lambda x, l: _run(x, l, decay)[0]), (torch.float64, lambda x, l: _plain(x, l, decay))):
        ls = [{n: cast(t, dt) for n, t in p.items()} for p in layers]
        xx = cast(x, dt)
        y = fn(xx, ls)
        leaves = [xx] + [t for p in ls for t in p.values()]
        got = [y.detach()] + list(torch.autograd.grad(y, leaves, gy.to(dtype).cuda().to(dt)))
        if dt is dtype:
            mine = got
    for i, (a, b) in enumerate(zip(mine, got)):
        err = ((a.double() - b).norm() / b.norm()).item()
        assert err <= (2e-4 if dtype == torch.float32 else 2.0 ** -5), (i, err)


def test_prompt_and_tokens():
    """Layer states of a prompt, then token by token: the rows of the whole sequence."""
    from hclsm_amd.kernels import linear_attention_step, residual_rms_norm
    g = torch.Generator().manual_seed(2)
    B, L, P = 2, 40, 33
    x = torch.randn(B, L, D, generator=g).cuda()
    layers = [{n: t.cuda() for n, t in p.items()} for p in _weights(g)]
    decay = -torch.tensor([0.0, 0.01, 0.1, 0.5, 0.002, 3.0]).cuda()
    with torch.no_grad():
        whole, ends = _run(x, layers, decay)
        y, states = _run(x[:, :P], layers, decay)
        assert ((y - whole[:, :P]).norm() / y.norm()).item() <= 1e-5
        for t in range(P, L):
            z, h = x[:, t], torch.zeros(B, D, device="cuda")
            for p, s in zip(layers, states):
                n, h = residual_rms_norm(z, h, p["w"])
                q, k, v = (a[:, 0] for a in _split((n @ p["qkv"])[:, None], B, 1))
                z = linear_attention_step(q, k, v, decay, s).reshape(B, H * DV) @ p["o"]
            n, h = residual_rms_norm(z, h)
            assert ((n - whole[:, t]).norm() / n.norm()).item() <= 2e-5, t
        for s, e in zip(states, ends):
            assert ((s - e).norm() / e.norm()).item() <= 2e-5


def test_eight_bit_input_of_a_projection():
    """y8 * scale against the norm in the input's type, through one projection: half a step of e4m3, 2^-4 of a value, at most."""
    from hclsm_amd.kernels import residual_rms_norm, residual_rms_norm_fp8
    g = torch.Generator().manual_seed(3)
    x, r, w = torch.randn(70, 256, generator=g).cuda(), torch.randn(70, 256, generator=g).cuda(), torch.rand(256, generator=g).cuda()
    W = torch.randn(256, 64, generator=g).cuda()
    y, h = residual_rms_norm(x, r, w)
    for group in (None, 64):
        y8, scale, h8 = residual_rms_norm_fp8(x, r, w, group=group)
        back = (y8.float().reshape(70, -1, group or 256) * scale[..., None]).reshape(70, 256)
        assert torch.equal(h, h8)
        assert ((back @ W - y @ W).norm() <= (2.0 ** -4 * y.abs() @ W.abs()).norm())
