"""Refusals of residual_rms_norm and residual_rms_norm_fp8 (CPU: nothing is launched)."""

from __future__ import annotations

import ctypes
import importlib

import pytest
import torch

from hclsm_amd.kernels import residual_rms_norm, residual_rms_norm_fp8

F = importlib.import_module("hclsm_amd.kernels.residual_norm")


def _meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_cpu_tensors_are_refused():
    x = torch.randn(2, 8)
    for f in (residual_rms_norm, residual_rms_norm_fp8):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            f(x)


def test_accepted():
    h = torch.bfloat16
    F._check("f", _meta(5), None, None, 0.0)
    F._check("f", _meta(2, 3, 16384, dtype=h), _meta(2, 3, 16384, dtype=h), _meta(16384), 1e-6)
    F._check("f", _meta(0, 8, dtype=h), _meta(0, 8), _meta(8, dtype=h), 1e-6)


@pytest.mark.parametrize("err, args", [
    (ValueError, (_meta(), None, None, 0.0)), (TypeError, (_meta(2, 8, dtype=torch.float64), None, None, 0.0)),
    (ValueError, (_meta(2, 0), None, None, 0.0)), (ValueError, (_meta(2, 16385), None, None, 0.0)),
    (ValueError, (_meta(2, 8), _meta(2, 9), None, 0.0)), (ValueError, (_meta(2, 8), _meta(1, 8), None, 0.0)),
    (TypeError, (_meta(2, 8), _meta(2, 8, dtype=torch.bfloat16), None, 0.0)),
    (TypeError, (_meta(2, 8, dtype=torch.bfloat16), _meta(2, 8, dtype=torch.float16), None, 0.0)),
    (ValueError, (_meta(2, 8), None, _meta(9), 0.0)), (ValueError, (_meta(2, 8), None, _meta(8, dtype=torch.float64), 0.0)),
    (ValueError, (_meta(2, 8), None, None, -1.0)), (ValueError, (_meta(2, 8), None, None, float("nan"))),
    (ValueError, (_meta(2, 8), None, None, float("inf"))),
])
def test_refusals(err, args):
    with pytest.raises(err):
        F._check("f", *args)


def test_abi_refusals_before_launch():
    from hclsm_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("libhclsm_amd.so not built")
    L, P = _lib.lib(), 256    # a stand-in address: every call below returns before anything is launched
    base = dict(x=P, r=P, w=P, h=P, gy=P, gh=P, y=P, h_out=P, scale=P, dx=P, dr=P, dw=P, x_sr=64, r_sr=64, h_sr=64, gy_sr=64,
                gh_sr=64, rows=4, D=64, eps=1e-6, dtype=1, stream_dtype=1, w_dtype=0)

    def block(**kw):
        b = _lib.HclsmResidualNorm()
        for n, v in {**base, **kw}.items():
            setattr(b, n, v)
        return ctypes.byref(b)

    for f in (lambda b: L.hclsm_residual_norm_forward(b, None), lambda b: L.hclsm_residual_norm_fp8(b, None),
              lambda b: L.hclsm_residual_norm_backward(b, P, 1 << 20, None)):
        assert f(None) == -1
        assert f(block(rows=-1)) == -2 and f(block(D=0)) == -2 and f(block(eps=-1.0)) == -2 and f(block(eps=float("nan"))) == -2
        assert f(block(dtype=3)) == -3 and f(block(stream_dtype=2)) == -3 and f(block(w_dtype=3)) == -3
        assert f(block(D=16385)) == -4
    fwd, fp8 = L.hclsm_residual_norm_forward, L.hclsm_residual_norm_fp8
    assert fwd(block(x=None), None) == -1 and fwd(block(y=None), None) == -1 and fwd(block(rows=0), None) == 0
    assert fp8(block(scale=None), None) == -1 and fp8(block(group=48), None) == -4 and fp8(block(group=128), None) == -2
    assert fp8(block(group=32, x=P + 2), None) == -4
    bwd = L.hclsm_residual_norm_backward
    assert bwd(block(h=None), P, 1 << 20, None) == -1 and bwd(block(), None, 0, None) == -1 and bwd(block(), P, 8, None) == -2
    assert bwd(block(), P + 4, 1 << 20, None) == -4
    assert bwd(block(rows=0, dw=None), None, 0, None) == 0
    ws = L.hclsm_residual_norm_backward_workspace
    assert ws(5000, 64) == 1024 * 64 * 4 and ws(0, 64) == 0 and ws(-1, 64) == -2 and ws(5, 0) == -2 and ws(5, 1 << 20) == -4
