"""Oracle: norms and rotations of heads, and cross attention, in float64.  TEST INFRASTRUCTURE ONLY.

  * rotate: pair i of a head's first rot elements times amp * exp(i * position * frequency_i)
    (the rotation of the vision encoder's heads, perception/vision_encoder.py:171-259, in both pair layouts);
  * norm_rotate / norm_rotate_grads: the root-mean-square norm of each head and its rotation, and their gradients;
  * cross_attention / cross_attention_grads: softmax attention of queries against keys of another length with shared
    key heads, live keys given as a boolean (B, Lk) array; a query without a live key gives zeros
    (the core of nn.MultiheadAttention with learned queries, dynamics/level2_goal.py:50-63).
"""

from __future__ import annotations

import numpy as np


def pair_columns(rot, layout):
    i = np.arange(rot // 2)
    return (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)


def rotate(x, pos, freq, amp=1.0, layout="half", back=False):
    """x (B, L, H, dh), pos (L,) or (B, L), freq (rot / 2,).  back: the transposed map (its gradient)."""
    x = np.asarray(x, np.float64)
    a, b = pair_columns(2 * len(freq), layout)
    pos = np.asarray(pos, np.float64)
    pos = pos[None] if pos.ndim == 1 else pos
    turn = amp * np.exp((-1j if back else 1j) * pos[:, :, None, None] * np.asarray(freq, np.float64))
    z = (x[..., a] + 1j * x[..., b]) * turn
    y = x.copy()
    y[..., a], y[..., b] = z.real, z.imag
    return y


def norm_rotate(x, w, pos, freq, amp=1.0, layout="half", eps=1e-6):
    x = np.asarray(x, np.float64)
    n = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * w
    return n if freq is None else rotate(n, pos, freq, amp, layout)


def norm_rotate_grads(x, w, g, pos, freq, amp=1.0, layout="half", eps=1e-6):
    """(dx, dw) of sum(g * norm_rotate(x))."""
    x, g = np.asarray(x, np.float64), np.asarray(g, np.float64)
    r = 1.0 / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps)
    d = g if freq is None else rotate(g, pos, freq, amp, layout, back=True)
    n = x * r
    dn = d * w
    return r * (dn - n * np.mean(dn * n, -1, keepdims=True)), (d * n).sum((0, 1, 2))


def _weights(q, k, live, scale):
    """(B, H, Lq, Lk) softmax weights, zero rows where nothing is live; q, k (B, L, H, dh) of equal heads."""
    s = np.einsum("blhd,bmhd->bhlm", q, k) * scale
    s = np.where(live[:, None, None, :], s, -np.inf)
    top = s.max(-1, keepdims=True, initial=-np.inf)
    p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
    tot = p.sum(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        lse = np.where(tot > 0, np.log(np.where(tot > 0, tot, 1.0)) + np.where(np.isfinite(top), top, 0.0), -np.inf)
    return p / np.where(tot > 0, tot, 1.0), lse[..., 0]


def _prepared(q, k, v, live):
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    G = q.shape[2] // k.shape[2]
    dead = ~live[:, :, None, None]                    # what a masked key holds does not matter, NaN included
    k, v = np.where(dead, 0.0, k), np.where(dead, 0.0, v)
    return q, np.repeat(k, G, 2), np.repeat(v, G, 2), G


def cross_attention(q, k, v, live, scale=None):
    """(out (B, Lq, H, dh), lse (B, H, Lq))."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    q, k, v, _ = _prepared(q, k, v, live)
    p, lse = _weights(q, k, live, scale)
    return np.einsum("bhlm,bmhd->blhd", p, v), lse


def cross_attention_grads(q, k, v, live, g, scale=None):
    """(dq, dk, dv) of sum(g * out)."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    q, k, v, G = _prepared(q, k, v, live)
    g = np.asarray(g, np.float64)
    p, _ = _weights(q, k, live, scale)
    dv = np.einsum("bhlm,blhd->bmhd", p, g)
    dp = np.einsum("blhd,bmhd->bhlm", g, v)
    ds = p * (dp - (dp * p).sum(-1, keepdims=True)) * scale
    dq = np.einsum("bhlm,bmhd->blhd", ds, k)
    dk = np.einsum("bhlm,blhd->bmhd", ds, q)
    B, M, H, D = dk.shape
    return dq, dk.reshape(B, M, H // G, G, D).sum(3), dv.reshape(B, M, H // G, G, D).sum(3)
