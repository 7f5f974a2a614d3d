"""Elementwise error bounds of the cross-attention kernels, from the roundings they make (float64 on the CPU).

U = 2^-24 (float32), e = finfo(type).eps / 2 for the operands' type (0 for float32: no operand is rounded), flush =
2^-126: the exponential and the matrix unit give zero for results below the smallest normal float32, so a weight is off by
up to flush whatever its size, and so is a sum; tiny = half the smallest fp16 step (2^-25) or flush for the other types.  With w = p the softmax weights, per query row:
  score      |ds| <= dh U scale sum|q k|, the float32 sum of dh products in any order, and the argument of the
             exponential is rounded twice: 2 U |s| log2(e); the logarithm of the sum once more.
  weight     relative error rel = 2 max(score error) + (Lk / 4 + 40) U: exponential, running sum of Lk / 4 terms in
             sequence and its joining, rescaling by exponentials of differences; then e for the rounding to the operand.
  out        (rel + e + (Lk / 4 + 40) U) sum(p |v|) + e |out| + tiny sum|v|.
  delta      sum(g out) from the rounded out: e sum(|g| |out|) + the error of out + dh U.
  ds         p (error of dP + error of delta) + (2 rel + e) |ds| with |dP error| <= dh U sum|g v|; tiny for fp16.
  dq, dk     scale times the sum of |ds error| |k| (|q|) and (n + 40) U of the terms for n of them in sequence; e |dq|.
  dv         (2 rel + e) sum(p |g|), (n + 40) U, tiny sum|g|; e |dv|.

fine: weights and ds in two operands, the second one the rounding's rest: e^2 in place of e (tiny as before) but for the
rounding of the results, and delta from out and its rest: e^2 |out| in place of e |out|."""

from __future__ import annotations

import numpy as np
import torch

U = 2.0 ** -24


def bounds(q, k, v, live, g=None, scale=None, dtype=torch.float32, qk_units=0.0, fine=False):
    """Bounds for (out,) or (out, dq, dk, dv); qk_units: relative error of q and k themselves, in units of U.  All
    inputs float64, masked keys and dead queries finite."""
    e = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    end = torch.finfo(dtype).eps / 2
    e = e * e if fine else e
    rest = end * end if fine else end
    flush = 2.0 ** -126
    tiny = 2.0 ** -25 if dtype == torch.float16 else flush
    B, Lq, H, dh = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    scale = dh ** -0.5 if scale is None else scale
    k, v = np.where(live[:, :, None, None], k, 0), np.where(live[:, :, None, None], v, 0)
    kr, vr = np.repeat(k, G, 2), np.repeat(v, G, 2)
    A = np.abs
    s = np.einsum("blhd,bmhd->bhlm", q, kr) * scale
    sabs = np.einsum("blhd,bmhd->bhlm", A(q), A(kr)) * scale
    dead = ~live[:, None, None, :]
    sm = np.where(dead, -np.inf, s)
    top = sm.max(-1, keepdims=True, initial=-np.inf)
    top = np.where(np.isfinite(top), top, 0)
    p = np.exp(sm - top)
    tot = p.sum(-1, keepdims=True)
    p = p / np.where(tot > 0, tot, 1)
    lse = np.log(np.where(tot > 0, tot, 1)) + top
    err_s = (dh + 2 * qk_units) * U * sabs + 3 * U * np.maximum(A(np.where(dead, 0, s)), A(lse)) + 2 * U * A(lse)
    seq = (Lk / 4 + 40) * U
    rel = 2 * np.where(dead, 0, err_s).max(-1, keepdims=True, initial=0) + seq
    pv = np.einsum("bhlm,bmhd->blhd", p, A(vr))
    out = np.einsum("bhlm,bmhd->blhd", p, vr)
    rel_o = rel[..., 0].transpose(0, 2, 1)[..., None]
    b_sum = (rel_o + e + seq) * pv + tiny * (1 + A(vr).sum(1)[:, None])
    b_out = b_sum + end * A(out)
    if g is None:
        return (b_out * (1 + 4 * e),)
    dp = np.einsum("blhd,bmhd->bhlm", g, vr)
    dpabs = np.einsum("blhd,bmhd->bhlm", A(g), A(vr))
    delta = (g * out).sum(-1).transpose(0, 2, 1)[..., None]
    err_delta = ((A(g) * (b_sum + rest * A(out))).sum(-1) + (dh + 4) * U * (A(g) * pv).sum(-1)).transpose(0, 2, 1)[..., None]
    ds = p * (dp - delta)
    err_ds = p * (dh * U * dpabs + err_delta + 3 * U * (dpabs + A(delta))) * (1 + e) + (2 * rel + e) * A(ds)
    err_ds = np.where(dead, 0, err_ds + tiny + flush * (A(dp) + A(delta)))
    nk, nr = (Lk + 40) * U, (Lq * G + 40) * U

    def shared(t):
        return t.reshape(B, Lk, Hk, G, dh).sum(3)

    qe = qk_units * U
    b_dq = scale * np.einsum("bhlm,bmhd->blhd", err_ds + (nk + qe) * A(ds), A(kr))
    b_dk = scale * shared(np.einsum("bhlm,blhd->bmhd", err_ds + (nr + qe) * A(ds), A(q)))
    b_dv = shared(np.einsum("bhlm,blhd->bmhd", (2 * rel + e + nr) * p + np.where(dead, 0, tiny), A(g)))
    dq = scale * np.einsum("bhlm,bmhd->blhd", ds, kr)
    dk = scale * shared(np.einsum("bhlm,blhd->bmhd", ds, q))
    dv = shared(np.einsum("bhlm,blhd->bmhd", p, g))
    grow = 1 + 4 * e
    return (b_out * grow, b_dq * grow + end * A(dq) + tiny, b_dk * grow + end * A(dk) + tiny,
            b_dv * grow + end * A(dv) + tiny)


def assert_within(got, ref, bound, what):
    got = got.detach().double().cpu().numpy()
    assert got.shape == ref.shape, f"{what}: shape {got.shape}, want {ref.shape}"
    assert np.isfinite(got).all(), f"{what}: not finite"
    over = np.abs(got - ref) - bound
    assert (over <= 0).all(), (f"{what}: off by {np.abs(got - ref).max():.3e}, {over.max():.3e} over the bound at "
                               f"{np.unravel_index(over.argmax(), over.shape)}, {(over > 0).sum()} elements")
