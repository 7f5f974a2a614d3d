"""The oracle of linear attention and of the residual norm against closed forms and differences (CPU)."""

from __future__ import annotations

import numpy as np
import torch

from oracle import linear_attention as ol
from oracle import residual_norm as on


def _case(B=2, L=9, H=4, Hk=2, dk=3, dv=5, seed=0):
    r = np.random.default_rng(seed)
    q, k, v = r.normal(size=(B, L, H, dk)), r.normal(size=(B, L, Hk, dk)), r.normal(size=(B, L, Hk, dv))
    return q, k, v, np.array([0.0, -0.1, -2.0, -np.inf][:H]), r.normal(size=(B, H, dk, dv)), r


def test_linear_attention_by_pairs():
    """The sum over pairs of tokens, weighted by a^(t - s), and a^(t + 1) of the first state."""
    q, k, v, g, s0, _ = _case()
    out, s1 = ol.linear_attention(q, k, v, g, 0.7, s0)
    for h in range(4):
        a, kh, vh = np.exp(g[h]), k[:, :, h // 2], v[:, :, h // 2]
        age = np.subtract.outer(np.arange(9), np.arange(9))
        w = np.where(age >= 0, a ** np.maximum(age, 0), 0.0)
        ref = np.einsum("ts,btd,bsd,bse->bte", w, q[:, :, h], kh, vh)
        ref += (a ** np.arange(1, 10))[None, :, None] * np.einsum("btd,bde->bte", q[:, :, h], s0[:, h])
        assert np.allclose(out[:, :, h], 0.7 * ref, rtol=1e-12, atol=1e-12)
        end = a ** 9 * s0[:, h] + np.einsum("s,bsd,bse->bde", a ** np.arange(8.0, -1, -1), kh, vh)
        assert np.allclose(s1[:, h], end, rtol=1e-12, atol=1e-12)
    assert np.allclose(out[:, :, 3], 0.7 * (q[:, :, 3] * k[:, :, 1]).sum(-1, keepdims=True) * v[:, :, 1])    # no memory


def test_linear_attention_lengths_and_parts():
    q, k, v, g, s0, _ = _case()
    out, s1 = ol.linear_attention(q, k, v, g, 1.0, s0, lens=[4, 0])
    ref, e = ol.linear_attention(q[:1, :4], k[:1, :4], v[:1, :4], g, 1.0, s0[:1])
    assert np.array_equal(out[:1, :4], ref) and np.array_equal(s1[:1], e) and np.array_equal(s1[1], s0[1])
    assert not out[0, 4:].any() and not out[1].any()
    rest, end = ol.linear_attention(q[:, 4:], k[:, 4:], v[:, 4:], g, 1.0, ol.linear_attention(q[:, :4], k[:, :4], v[:, :4], g, 1.0, s0)[1])
    whole = ol.linear_attention(q, k, v, g, 1.0, s0)
    assert np.allclose(rest, whole[0][:, 4:]) and np.allclose(end, whole[1])


def test_linear_attention_grads_against_autograd():
    q, k, v, g, s0, r = _case()
    g = np.array([0.0, -0.1, -2.0, -50.0])
    go, gs = r.normal(size=(2, 9, 4, 5)), r.normal(size=s0.shape)
    for lens in (None, [9, 5]):
        t = [torch.tensor(x, requires_grad=True) for x in (q, k, v, s0)]
        a, loss = torch.exp(torch.tensor(g))[:, None, None], 0.0
        for b in range(2):
            S = t[3][b]
            for i in range(9 if lens is None else lens[b]):
                S = a * S + t[1][b, i].repeat_interleave(2, 0)[:, :, None] * t[2][b, i].repeat_interleave(2, 0)[:, None, :]
                loss = loss + (0.3 * torch.matmul(t[0][b, i][:, None], S)[:, 0] * torch.tensor(go[b, i])).sum()
            loss = loss + (S * torch.tensor(gs[b])).sum()
        ref = torch.autograd.grad(loss, t)
        got = ol.linear_attention_grads(q, k, v, g, 0.3, go, s0, gs, lens)
        for x, y in zip(got, ref):
            assert np.allclose(x, y.numpy(), rtol=1e-11, atol=1e-11)


def test_residual_norm_against_autograd():
    r = np.random.default_rng(1)
    h, w, gy, gh = r.normal(size=(3, 7)), r.normal(size=7), r.normal(size=(3, 7)), r.normal(size=(3, 7))
    th, tw = torch.tensor(h, requires_grad=True), torch.tensor(w, requires_grad=True)
    y = torch.nn.functional.rms_norm(th, (7,), tw, 1e-3)
    assert np.allclose(on.rms_norm(h, w, 1e-3), y.detach().numpy(), rtol=1e-12)
    ref = torch.autograd.grad((y, th * 1.0), (th, tw), (torch.tensor(gy), torch.tensor(gh)))
    for a, b in zip(on.rms_norm_grads(h, gy, gh, w, 1e-3), ref):
        assert np.allclose(a, b.numpy(), rtol=1e-11)
    assert np.allclose(on.scales([[0.0, 0.0, -448.0, 1.0]], 2), [[2.0 ** -100 / 448, 1.0]])
    assert np.allclose(on.scales([[0.0, 0.0, -448.0, 1.0]]), [[1.0]])
