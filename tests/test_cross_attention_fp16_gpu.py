"""float16 cross attention away from unit gradients and short keys, against oracle/heads.py (float64).

What is rounded to float16 besides the results is rounded in a range of its own, so an error in a result is that of some
sums of independent relative roundings:
  rms     ds and the result each round with the same relative step, so the rms error of a gradient is sqrt(2) times the
          rms of rounding the float64 gradient to float16 (a sum of terms of either sign carries the terms' relative rms), and
          as much again only if something else is lost.  At most 2 is allowed.
  bound   elementwise that of cross_attention_bounds.py, for gradients 2^K times as large and divided by 2^K: the formulas are
          linear in g, and its allowance for subnormal roundings, 2^-25 in each ds, stands for values near one.  K is 10 - log2(max|ds|),
          since a row's or key's largest ds is rounded at 2^10 or above: a step of 2^-35 of it.  K is at most 12 for dv, whose
          weights are rounded at 2^12 times their size.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cross_attention_bounds import bounds
from oracle import heads as oh

pytestmark = pytest.mark.gpu


def _np(t):
    return t.detach().double().cpu().numpy()


def _case(B, Lq, Lk, H, Hk, dh, g_size, v_size, seed):
    r = torch.Generator().manual_seed(seed)
    rnd = lambda size, *s: (size * torch.randn(*s, generator=r)).half()
    return rnd(1, B, Lq, H, dh), rnd(1, B, Lk, Hk, dh), rnd(v_size, B, Lk, Hk, dh), rnd(g_size, B, Lq, H, dh)


def _most_ds(q, k, v, live, g, scale):
    """The largest magnitude of p (dP - delta)."""
    G = q.shape[2] // k.shape[2]
    k, v = np.repeat(k, G, 2), np.repeat(v, G, 2)
    p, _ = oh._weights(q, k, live, scale)
    dp = np.einsum("blhd,bmhd->bhlm", g, v)
    return np.abs(p * (dp - (p * dp).sum(-1, keepdims=True))).max()


def _rms(t):
    return np.sqrt(np.mean(t * t))


def _check(case, what, scale=None, live=None, names=("dq", "dk"), **masks):
    from hclsm_amd.kernels import cross_attention
    q, k, v, g = case
    ins = [t.cuda().requires_grad_() for t in (q, k, v)]
    out = cross_attention(*ins, scale=scale, **masks)
    grads = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, ins, g.cuda())))
    vals, gn = [_np(t) for t in (q, k, v)], _np(g)
    s = q.shape[-1] ** -0.5 if scale is None else scale
    live = np.ones((q.shape[0], k.shape[1]), bool) if live is None else live
    vals[1], vals[2] = (np.where(live[:, :, None, None], t, 0) for t in vals[1:])
    refs = dict(zip(("dq", "dk", "dv"), oh.cross_attention_grads(*vals, live, gn, s)))
    K = int(np.floor(10 - np.log2(_most_ds(*vals, live, gn, s))))
    bs = {}
    for name in names:
        K = min(K, 12) if name == "dv" else K
        if K not in bs:
            bs[K] = dict(zip(("out", "dq", "dk", "dv"), bounds(*vals, live, gn * 2.0 ** K, s, torch.float16)))
        got, ref = _np(grads[name]), refs[name]
        assert np.isfinite(got).all(), f"{what} {name}: not finite"
        over = np.abs(got - ref) - (bs[K][name] * 2.0 ** -K + 2.0 ** -25)
        assert (over <= 0).all(), f"{what} {name}: {over.max():.3e} over the bound"
        own = _rms(np.float64(np.float16(ref)) - ref)
        err = _rms(got - ref)
        print(f"{what} {name}: rms error {err:.3e}, {err / own:.2f} times its rounding", flush=True)
        assert err <= 2 * own, f"{what} {name}: rms error {err:.3e}, rounding {own:.3e}"


TILED = [(1, 64, 4096, 2, 2, 64), (1, 64, 32768, 1, 1, 64), (2, 70, 1003, 4, 2, 80), (1, 130, 700, 1, 1, 128),
         (1, 40, 2000, 2, 1, 256), (2, 33, 300, 3, 1, 32), (1, 200, 30, 2, 2, 96)]
FEW = [(2, 1, 4096, 8, 2, 64), (1, 4, 32768, 2, 1, 64), (2, 32, 196, 3, 3, 64), (1, 9, 3000, 2, 1, 128), (1, 7, 900, 4, 1, 96)]


@pytest.mark.parametrize("g_size", [1.0, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("shape", TILED + FEW)
def test_gradients_of_any_size(shape, g_size):
    _check(_case(*shape, g_size, 1.0, 41), f"{shape} g {g_size}")


@pytest.mark.parametrize("shape", [(1, 64, 32768, 2, 2, 64), (1, 40, 131072, 1, 1, 32), (1, 4, 131072, 2, 1, 64),
                                   (1, 70, 40000, 1, 1, 256)])
def test_weights_of_long_keys(shape):
    """Weights near 2^-17, of which float16 holds some 7 bits."""
    _check(_case(*shape, 30.0, 1.0, 46), f"{shape} long", names=("dq", "dk", "dv"))


@pytest.mark.parametrize("shape", TILED + FEW)
def test_gradients_of_the_values(shape):
    _check(_case(*shape, 1.0, 1.0, 47), f"{shape}", names=("dv",))


@pytest.mark.parametrize("shape", [(1, 64, 40, 2, 2, 64), (1, 64, 300, 2, 2, 128), (2, 8, 40, 4, 2, 64), (1, 64, 30, 1, 1, 32)])
def test_scores_gradients_past_float16_with_results_inside(shape):
    """v of 2000 and g of 200: ds up to some 10^5, past 65504, and results of hundreds."""
    case = _case(*shape, 200.0, 2000.0, 42)
    vals = [_np(t) for t in case[:3]]
    assert _most_ds(*vals, np.ones((shape[0], shape[2]), bool), _np(case[3]), 1e-3) > 65504 / (4 if shape[2] > 100 else 1)
    _check(case, f"{shape} large", scale=1e-3)


@pytest.mark.parametrize("shape", [(1, 64, 1500, 2, 2, 64), (1, 8, 1500, 2, 2, 64), (1, 96, 600, 1, 1, 128)])
@pytest.mark.parametrize("order", ["up", "down"])
def test_gradients_that_grow_along_the_keys_and_rows(shape, order):
    """v grows (or shrinks) by 2^16 along the keys and g by 2^10 along the rows: the factor is lowered on the way."""
    q, k, v, g = _case(*shape, 1e-2, 1.0, 43)
    along = lambda t, octaves: (t.double() * 2.0 ** (octaves * torch.linspace(-1, 0, t.shape[1], dtype=torch.float64))[:, None, None]).half()
    v, g = along(v, 16) * 100, along(g, 10) * 100
    if order == "down":
        k, v, q, g = (t.flip(1).contiguous() for t in (k, v, q, g))
    _check((q, k, v, g), f"{shape} {order}")


@pytest.mark.parametrize("shape", [(3, 40, 500, 2, 1, 64), (3, 5, 500, 2, 1, 64)])
def test_masked_keys_do_not_move_the_factor(shape):
    """Infinities and NaN in masked keys, an empty row: live results as exact as without them."""
    q, k, v, g = _case(*shape, 1e-3, 1.0, 44)
    r = np.random.default_rng(45)
    pad = r.random(k.shape[:2]) < 0.3
    pad[1] = True
    v[torch.tensor(pad)], k[torch.tensor(pad)] = float("inf"), float("nan")
    k[2][torch.tensor(pad[2])] = 60000.0
    _check((q, k, v, g), f"{shape} masked", live=~pad, key_padding_mask=torch.tensor(pad).cuda())


@pytest.mark.parametrize("gap", [14.0, 18.0, 21.0])
@pytest.mark.parametrize("where", [0, -1])
@pytest.mark.parametrize("shape", [(1, 64, 32768, 1, 1, 64), (1, 2, 32768, 2, 1, 64), (1, 1, 50000, 4, 1, 128), (1, 70, 9000, 1, 1, 256)])
def test_many_weights_far_below_the_largest(shape, where, gap):
    """One key `gap` above all others with a value near zero: the others are what the output is made of.  Its weight is at
    least 2^11, so a rounding of the smallest ones is off by at most 2^-36 of the softmax.  One batch row expanded to 800, so
    that no row's keys are split over workgroups (each with a largest weight of its own)."""
    from hclsm_amd.kernels import cross_attention
    B, Lq, Lk, H, Hk, dh = shape
    q, k, v, _ = _case(*shape, 1.0, 1.0, 48)
    q, k, v = 0.3 * q, 0.3 * k, 1 + 0.1 * v
    q[..., 0], k[..., 0] = 16, 0
    k[:, where], v[:, where] = 0, 0.01
    k[:, where, :, 0] = gap / (16 * dh ** -0.5)
    with torch.no_grad():
        rows = cross_attention(*(t.cuda().expand(800, -1, -1, -1) for t in (q, k, v)))
        assert torch.equal(rows, rows[:1].expand(800, -1, -1, -1))
        got = _np(rows[:1])
    vals, live = [_np(t) for t in (q, k, v)], np.ones((B, Lk), bool)
    ref, _ = oh.cross_attention(*vals, live)
    (b,) = bounds(*vals, live, None, None, torch.float16)
    least = 1 + np.abs(vals[2]).sum(1)[:, None].repeat(H // Hk, 2)
    over = np.abs(got - ref) - (b - (1 - 2.0 ** -11) * 2.0 ** -25 * least + 2.0 ** -25)
    print(f"{shape} gap {gap}: off by {np.abs(got - ref).max():.2e} of {np.abs(ref).max():.2e}", flush=True)
    assert (over <= 0).all(), f"{over.max():.3e} over the bound"
