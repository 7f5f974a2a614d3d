"""Refusals of the norm and rotation of heads, and the plan's frequencies (CPU: nothing is launched)."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from hclsm_amd.kernels import RotaryPlan, qk_norm_rotary, rotary_embedding


def test_plan_frequencies():
    p = RotaryPlan(8, device="cpu")
    assert torch.allclose(p.inv_freq, 10000.0 ** (-torch.arange(4, dtype=torch.float64) / 4), rtol=1e-15)
    assert torch.allclose(RotaryPlan(8, scaling="linear", factor=4.0, device="cpu").inv_freq, p.inv_freq / 4)
    ntk = RotaryPlan(8, scaling="ntk", factor=4.0, device="cpu").inv_freq
    assert ntk[0] == 1 and math.isclose(ntk[-1].item(), p.inv_freq[-1].item() / 4, rel_tol=1e-12)
    y = RotaryPlan(128, scaling="yarn", factor=8.0, original_length=4096, device="cpu")
    full = RotaryPlan(128, device="cpu").inv_freq
    turns = full * 4096 / (2 * math.pi)
    assert torch.equal(y.inv_freq[turns > 40], full[turns > 40])
    assert torch.allclose(y.inv_freq[turns < 0.8], full[turns < 0.8] / 8)
    assert (y.inv_freq <= full).all() and (y.inv_freq >= full / 8 * (1 - 1e-12)).all()
    assert math.isclose(y.amplitude, 0.1 * math.log(8) + 1)
    own = RotaryPlan(4, inv_freq=torch.tensor([0.5, 0.25]), amplitude=2.0, device="cpu")
    assert own.inv_freq.tolist() == [0.5, 0.25] and own.amplitude == 2.0


@pytest.mark.parametrize("kw", [dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=258), dict(rot_dim=8, layout="x"),
                                dict(rot_dim=8, scaling="x"), dict(rot_dim=8, scaling="yarn", factor=2.0),
                                dict(rot_dim=8, base=1.0), dict(rot_dim=8, factor=0.0),
                                dict(rot_dim=8, inv_freq=torch.ones(3)),
                                dict(rot_dim=8, inv_freq=torch.full((4,), float("nan"))),
                                dict(rot_dim=8, inv_freq=torch.ones(4), scaling="linear"),
                                dict(rot_dim=8, scaling="yarn", factor=2.0, original_length=64, beta_fast=1.0)])
def test_plan_refusals(kw):
    with pytest.raises(ValueError):
        RotaryPlan(device="cpu", **kw)


def test_cpu_tensors_are_refused():
    plan = RotaryPlan(8, device="cpu")
    x = torch.randn(1, 2, 3, 8)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        rotary_embedding(x, plan)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        qk_norm_rotary(x, x, None, None, plan)


def _meta(*shape, dtype=torch.float32):
    """Checks run before anything is launched: shapes and types are all they look at."""
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("err, call", [
    (ValueError, lambda f, p: f._check_heads("f", "x", _meta(2, 3, 8))),
    (TypeError, lambda f, p: f._check_heads("f", "x", _meta(1, 2, 3, 8, dtype=torch.float64))),
    (ValueError, lambda f, p: f._check_heads("f", "x", _meta(1, 2, 3, 257))),
    (ValueError, lambda f, p: f._check_plan("f", p, 6)),
    (TypeError, lambda f, p: f._check_plan("f", 8, 8)),
    (TypeError, lambda f, p: f._check_positions("f", "p", _meta(2), _meta(1, 2, 3, 8))),
    (ValueError, lambda f, p: f._check_positions("f", "p", _meta(3, dtype=torch.int64), _meta(1, 2, 3, 8))),
    (ValueError, lambda f, p: f._check_positions("f", "p", _meta(2, 1, dtype=torch.int64), _meta(1, 2, 3, 8))),
])
def test_refusals(err, call):
    from hclsm_amd.kernels import norm_rotary
    with pytest.raises(err):
        call(norm_rotary, RotaryPlan(8, device="cpu"))


def test_abi_refusals_before_launch():
    from hclsm_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("libhclsm_amd.so not built")
    L, P = _lib.lib(), 256    # a stand-in address: every call below returns before anything is launched

    def heads(**kw):
        h = _lib.HclsmHeads(P, P, P, None, None, None, 128, 64, 32, 128, 64, 32, 0, 0, 2, 2, 2, 0, 0)
        for n, v in kw.items():
            setattr(h, n, v)
        return ctypes.byref(h)

    def fwd(q=None, k=None, dh=32, rot=32, layout=0, turns=P, norm=1, dtype=1):
        return L.hclsm_norm_rotary_forward(heads() if q is None else q, k, dh, rot, layout, turns, 1.0, 1e-6, norm,
                                           dtype, None)

    assert L.hclsm_norm_rotary_forward(None, None, 32, 32, 0, P, 1.0, 1e-6, 1, 1, None) == -1
    assert fwd(q=heads(x=None)) == -1 and fwd(q=heads(y=None)) == -1 and fwd(turns=None) == -1
    assert fwd(k=heads(x=None)) == -1
    assert fwd(dh=0) == -2 and fwd(rot=33) == -2 and fwd(rot=34) == -2 and fwd(q=heads(B=-1)) == -2
    assert fwd(dtype=3) == -3 and fwd(q=heads(pos=P, pos_dtype=2)) == -3 and fwd(q=heads(w=P, w_dtype=3)) == -3
    assert fwd(dh=257) == -4 and fwd(q=heads(B=1 << 30, L=4)) == -4 and fwd(layout=2) == -5
    assert fwd(q=heads(B=0)) == 0                                     # nothing to do
    ws = L.hclsm_norm_rotary_backward_workspace
    assert ws(32, 1) == 1024 * 32 * 4 and ws(32, 2) == 2 * ws(32, 1) and ws(0, 1) == -2 and ws(32, 3) == -2

    def bwd(q, ws_ptr, n):
        return L.hclsm_norm_rotary_backward(q, None, 32, 32, 0, P, 1.0, 1e-6, 1, ws_ptr, n, None)

    assert bwd(heads(g=None), P, 1 << 20) == -1
    assert bwd(heads(w=P, gw=P), P, 4) == -2 and bwd(heads(w=P, gw=P), None, 1 << 20) == -1
