"""Refusals of cross_attention (CPU: nothing is launched)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from hclsm_amd.kernels import cross_attention
from hclsm_amd.kernels import cross_attention as _fn  # noqa: F401  (the package exports the function)


def _module():
    import importlib
    return importlib.import_module("hclsm_amd.kernels.cross_attention")


def _meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


def _check(q=(2, 3, 4, 16), k=(2, 5, 2, 16), v=None, mask=None, klens=None, qlens=None, scale=0.25, dt=torch.float32,
           kdt=None):
    _module()._check(_meta(*q, dtype=dt), _meta(*k, dtype=kdt or dt), _meta(*(v or k), dtype=kdt or dt), mask, klens,
                     qlens, scale)


def test_cpu_tensors_are_refused():
    x = torch.randn(1, 2, 3, 16)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        cross_attention(x, x, x)


def test_accepted():
    _check()
    _check(q=(2, 0, 4, 256), k=(2, 0, 1, 256))
    _check(mask=_meta(2, 5, dtype=torch.bool), klens=_meta(2, dtype=torch.int32), qlens=_meta(2, dtype=torch.int64))


@pytest.mark.parametrize("err, kw", [
    (ValueError, dict(q=(3, 4, 16))), (ValueError, dict(k=(2, 5, 3, 16))), (ValueError, dict(k=(2, 5, 0, 16))),
    (ValueError, dict(k=(1, 5, 2, 16))), (ValueError, dict(k=(2, 5, 2, 8))), (ValueError, dict(v=(2, 6, 2, 16))),
    (ValueError, dict(q=(2, 3, 4, 12), k=(2, 5, 2, 12))), (ValueError, dict(q=(2, 3, 4, 264), k=(2, 5, 2, 264))),
    (TypeError, dict(dt=torch.float64)), (TypeError, dict(kdt=torch.bfloat16)),
    (ValueError, dict(mask=_meta(2, 4, dtype=torch.bool))), (ValueError, dict(klens=_meta(3, dtype=torch.int32))),
    (TypeError, dict(klens=_meta(2))), (TypeError, dict(qlens=_meta(2, dtype=torch.int16))),
    (ValueError, dict(qlens=_meta(2, 1, dtype=torch.int64))),
    (ValueError, dict(scale=0.0)), (ValueError, dict(scale=-1.0)), (ValueError, dict(scale=float("nan"))),
    (ValueError, dict(scale=float("inf"))),
])
def test_refusals(err, kw):
    with pytest.raises(err):
        _check(**kw)


def test_abi_refusals_before_launch():
    from hclsm_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("libhclsm_amd.so not built")
    L, P = _lib.lib(), 4096    # a stand-in address: every call below returns before anything is launched

    def call(backward=False, ws=P, ws_bytes=1 << 40, **kw):
        x = _lib.HclsmCrossAttention(B=2, Lq=3, Lk=5, H=4, Hk=2, dh=16, scale=0.25, dtype=1)
        for n in ("q", "k", "v", "g", "out", "lse", "dq", "dk", "dv"):
            setattr(x, n, P)
        for n in ("q", "k", "v", "g"):
            for s in ("sb", "sl", "sh"):
                setattr(x, f"{n}_{s}", 64)
        for n, val in kw.items():
            setattr(x, n, val)
        f = L.hclsm_cross_attention_backward if backward else L.hclsm_cross_attention_forward
        return f(ctypes.byref(x), ws, ws_bytes, None)

    assert L.hclsm_cross_attention_forward(None, None, 0, None) == -1
    for n in ("q", "k", "v", "out"):
        assert call(**{n: None}) == -1
    for n in ("g", "lse", "dk", "dv"):
        assert call(True, **{n: None}) == -1
    assert call(True, dq=None, dk=None, dv=None) == 0                   # nothing wanted
    assert call(True, ws=None, Lq=40) == -1 and call(True, ws_bytes=4, Lq=40) == -2
    assert call(ws=None, Lk=5000) == -1 and call(ws_bytes=4, Lk=5000) == -2          # keys split over workgroups
    for kw in (dict(B=-1), dict(Hk=3), dict(Hk=0), dict(dh=0), dict(scale=0.0), dict(scale=float("nan")),
               dict(Lq=1 << 31)):
        assert call(**kw) == -2, kw
    for kw in (dict(dtype=3), dict(key_lens_dtype=2), dict(query_lens_dtype=-1)):
        assert call(**kw) == -3, kw
    for kw in (dict(dh=12), dict(dh=264), dict(q=P + 8), dict(k_sl=60), dict(v_sh=4), dict(out=P + 8),
               dict(Lq=(1 << 31) - 1), dict(Lk=(1 << 31) - 1), dict(B=1 << 30)):
        assert call(**kw) == -4, kw
    assert call(B=0) == 0 and call(Lq=0) == 0 and call(True, B=0) == 0
    ws = L.hclsm_cross_attention_workspace
    assert ws(2, 3, 5, 4, 2, 16, 1, 0) == 0 and ws(2, 40, 5, 4, 2, 16, 1, 1) > 0 and ws(2, 3, 5000, 4, 2, 16, 1, 0) > 0
    assert ws(2, 3, 5, 4, 2, 12, 1, 1) == -4 and ws(2, 3, 5, 4, 3, 16, 1, 0) == -2


def test_abi_refuses_unaligned_workspaces_and_scales_past_float32():
    from hclsm_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("libhclsm_amd.so not built")
    L, P = _lib.lib(), 4096
    x = _lib.HclsmCrossAttention(B=2, Lq=40, Lk=5000, H=4, Hk=2, dh=16, scale=0.25, dtype=1)
    for n in ("q", "k", "v", "g", "out", "lse", "dq", "dk", "dv"):
        setattr(x, n, P)
    big = 1 << 40
    assert L.hclsm_cross_attention_forward(ctypes.byref(x), P + 4, big, None) == -4
    assert L.hclsm_cross_attention_backward(ctypes.byref(x), P + 8, big, None) == -4
    x.scale = 2.5e38      # times log2(e): past float32
    assert L.hclsm_cross_attention_forward(ctypes.byref(x), P, big, None) == -2
    assert L.hclsm_cross_attention_backward(ctypes.byref(x), P, big, None) == -2


@pytest.mark.parametrize("scale", [1e-46, 1e39, 2.5e38])
def test_scales_that_float32_does_not_hold(scale):
    with pytest.raises(ValueError, match="scale"):
        _check(scale=scale)
