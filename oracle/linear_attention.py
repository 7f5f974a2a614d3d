"""Oracle: linear attention with a decay for each head, in float64, token by token.  TEST INFRASTRUCTURE ONLY.

S_t = a_h S_{t-1} + k_t v_t^T, out_t = scale q_t^T S_t with a_h = exp(log_decay_h), and its gradients by the adjoint
recurrence D_t = scale q_t g_t^T + a_h D_{t+1}.  Rows of shared key heads repeat for the heads that read them.
"""

from __future__ import annotations

import numpy as np


def _f64(*ts):
    return tuple(None if t is None else np.asarray(t, np.float64) for t in ts)


def _heads(t, H):
    return np.repeat(t, H // t.shape[2], axis=2)


def linear_attention(q, k, v, log_decay, scale, state=None, lens=None):
    """q (B, L, H, dk), k, v (B, L, Hk, dk / dv), state (B, H, dk, dv); lens (B,) live tokens.  (out, last state)."""
    q, k, v, g = _f64(q, k, v, log_decay)
    B, L, H, dk = q.shape
    dv = v.shape[3]
    S = np.zeros((B, H, dk, dv)) if state is None else np.array(state, np.float64)
    out = np.zeros((B, L, H, dv))
    a = np.exp(g)[:, None, None]
    for b in range(B):
        n = L if lens is None else min(max(int(lens[b]), 0), L)
        kb, vb = _heads(k[b:b + 1, :n], H)[0], _heads(v[b:b + 1, :n], H)[0]
        for t in range(n):
            S[b] = a * S[b] + kb[t][:, :, None] * vb[t][:, None, :]
            out[b, t] = scale * np.matmul(q[b, t][:, None, :], S[b])[:, 0]
    return out, S


def linear_attention_grads(q, k, v, log_decay, scale, g, state=None, gs=None, lens=None):
    """Gradients of sum(g out) + sum(gs state) for q, k, v and the first state."""
    q, k, v, ld, g = _f64(q, k, v, log_decay, g)
    B, L, H, dk = q.shape
    Hk, dv = k.shape[2], v.shape[3]
    a = np.exp(ld)[:, None, None]
    S0 = np.zeros((B, H, dk, dv)) if state is None else np.asarray(state, np.float64)
    dS = np.zeros((B, H, dk, dv)) if gs is None else np.array(gs, np.float64)
    dq, dk_, dv_ = np.zeros(q.shape), np.zeros((B, L, H, dk)), np.zeros((B, L, H, dv))
    for b in range(B):
        n = L if lens is None else min(max(int(lens[b]), 0), L)
        kb, vb = _heads(k[b:b + 1, :n], H)[0], _heads(v[b:b + 1, :n], H)[0]
        S = S0[b].copy()
        for t in range(n):
            S = a * S + kb[t][:, :, None] * vb[t][:, None, :]
            dq[b, t] = scale * np.matmul(S, g[b, t][:, :, None])[..., 0]
        D = dS[b]
        for t in range(n - 1, -1, -1):
            D = D + scale * q[b, t][:, :, None] * g[b, t][:, None, :]
            dk_[b, t] = np.matmul(D, vb[t][:, :, None])[..., 0]
            dv_[b, t] = np.matmul(kb[t][:, None, :], D)[:, 0]
            D = a * D
        dS[b] = D
    fold = lambda t: t.reshape(B, L, Hk, H // Hk, -1).sum(3)
    return dq, fold(dk_), fold(dv_), dS
