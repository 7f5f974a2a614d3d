"""Refusals of linear_attention and linear_attention_step (CPU: nothing is launched)."""

from __future__ import annotations

import ctypes
import importlib

import pytest
import torch

from hclsm_amd.kernels import linear_attention, linear_attention_step

F = importlib.import_module("hclsm_amd.kernels.linear_attention")


def _meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


def _check(q=(2, 3, 4, 16), k=(2, 3, 2, 16), v=(2, 3, 2, 24), g=(4,), gdt=torch.float32, scale=0.25, dt=torch.float32, vdt=None,
           token=False):
    F._check("f", _meta(*q, dtype=dt), _meta(*k, dtype=dt), _meta(*v, dtype=vdt or dt), _meta(*g, dtype=gdt), scale, token)


def test_cpu_tensors_are_refused():
    x, g = torch.randn(1, 2, 3, 16), torch.zeros(3)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        linear_attention(x, x, x, g)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        linear_attention_step(x[:, 0], x[:, 0], x[:, 0], g, torch.zeros(1, 3, 16, 16))


def test_accepted():
    _check()
    _check(q=(2, 0, 4, 256), k=(2, 0, 1, 256), v=(2, 0, 1, 8))
    _check(q=(2, 4, 16), k=(2, 2, 16), v=(2, 2, 24), token=True)


@pytest.mark.parametrize("err, kw", [
    (ValueError, dict(q=(3, 4, 16))), (ValueError, dict(k=(2, 3, 3, 16), v=(2, 3, 3, 16))),
    (ValueError, dict(k=(2, 3, 0, 16), v=(2, 3, 0, 16))), (ValueError, dict(k=(2, 4, 2, 16))),
    (ValueError, dict(k=(2, 3, 2, 8))), (ValueError, dict(v=(2, 3, 1, 16))), (ValueError, dict(v=(2, 3, 2, 12))),
    (ValueError, dict(v=(2, 3, 2, 264))), (ValueError, dict(q=(2, 3, 4, 12), k=(2, 3, 2, 12))),
    (TypeError, dict(dt=torch.float64)), (TypeError, dict(vdt=torch.bfloat16)), (ValueError, dict(g=(2,))),
    (ValueError, dict(gdt=torch.float64)), (ValueError, dict(scale=0.0)), (ValueError, dict(scale=-1.0)),
    (ValueError, dict(scale=float("nan"))), (ValueError, dict(scale=float("inf"))), (ValueError, dict(token=True)),
    (ValueError, dict(q=(1 << 19, 1, 4, 16), k=(1 << 19, 1, 4, 16), v=(1 << 19, 1, 4, 16))),
])
def test_refusals(err, kw):
    with pytest.raises(err):
        _check(**kw)


def test_a_decay_that_learns_is_refused():
    q = _meta(2, 3, 4, 16)
    with pytest.raises(ValueError, match="no gradient"):
        F._check("f", q, q, q, torch.zeros(4, requires_grad=True), 1.0, False)


@pytest.mark.parametrize("err, t", [(TypeError, _meta(2)), (TypeError, _meta(2, dtype=torch.int16)),
                                    (ValueError, _meta(3, dtype=torch.int32)), (ValueError, _meta(2, 1, dtype=torch.int64))])
def test_index_refusals(err, t):
    with pytest.raises(err):
        F._check_index("f", "rows", t, 2)


@pytest.mark.parametrize("state", [
    _meta(2, 4, 16, 23), _meta(3, 4, 16, 24), _meta(2, 4, 16, 24, dtype=torch.bfloat16), _meta(4, 16, 24),
    _meta(2, 4, 24, 16).transpose(2, 3), _meta(1, 4, 16, 24).expand(2, 4, 16, 24), _meta(2, 1, 16, 24).expand(2, 4, 16, 24),
    _meta(2, 4, 16, 48)[..., :24], _meta(2, 8, 16, 24)[:, ::2],
])
def test_state_refusals(state):
    with pytest.raises(ValueError):
        F._check_state("f", state, 2, 4, 16, 24)


def test_state_views_accepted():
    F._check_state("f", _meta(2, 4, 16, 24), 2, 4, 16, 24)
    F._check_state("f", _meta(2, 8, 16, 24)[:, :4], 2, 4, 16, 24)
    F._check_state("f", _meta(9, 4, 16, 24)[::2], None, 4, 16, 24)


def test_abi_refusals_before_launch():
    from hclsm_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("libhclsm_amd.so not built")
    L, P = _lib.lib(), 256    # a stand-in address: every call below returns before anything is launched
    ws = L.hclsm_linear_attention_workspace
    assert ws(2, 1024, 6, 6, 64, 64, 1, 0) >= 0 and ws(64, 64, 16, 16, 64, 64, 1, 0) == 0
    assert ws(1, 1 << 16, 2, 2, 64, 64, 1, 0) > 0                  # split over time
    assert ws(-1, 4, 2, 2, 64, 64, 1, 0) == -2 and ws(1, 4, 3, 2, 64, 64, 1, 0) == -2 and ws(1, 4, 2, 2, 64, 64, 3, 0) == -3
    assert ws(1, 4, 2, 2, 60, 64, 1, 0) == -4 and ws(1, 4, 2, 2, 64, 264, 1, 0) == -4 and ws(1 << 20, 4, 2, 2, 64, 64, 1, 0) == -4

    def block(kind, **kw):
        b = kind()
        for n, v in kw.items():
            setattr(b, n, v)
        return ctypes.byref(b)

    base = dict(q=P, k=P, v=P, g=P, log_decay=P, out=P, dq=P, dk_out=P, dv_out=P, q_sb=64, q_sl=32, q_sh=16, k_sb=64, k_sl=32,
                k_sh=16, v_sb=64, v_sl=32, v_sh=16, g_sb=64, g_sl=32, g_sh=16, B=2, L=2, H=2, Hk=2, dk=16, dv=16, scale=0.25, dtype=1)
    for f in (L.hclsm_linear_attention_forward, L.hclsm_linear_attention_backward):
        run = lambda **kw: f(block(_lib.HclsmLinearAttention, **{**base, **kw}), P, 1 << 20, None)
        assert f(None, None, 0, None) == -1
        assert run(q=None) == -1 and run(k=None) == -1 and run(v=None) == -1 and run(log_decay=None) == -1
        assert run(B=-1) == -2 and run(H=3) == -2 and run(scale=0.0) == -2 and run(scale=float("nan")) == -2
        assert run(dtype=3) == -3 and run(seq_lens_dtype=2) == -3
        assert run(dk=20) == -4 and run(q=P + 8) == -4 and run(k_sl=36) == -4
        assert run(B=0) == 0 and run(H=0) == 0
    assert L.hclsm_linear_attention_forward(block(_lib.HclsmLinearAttention, **{**base, "out": None}), P, 1 << 20, None) == -1
    assert L.hclsm_linear_attention_forward(block(_lib.HclsmLinearAttention, **{**base, "out": P + 8}), P, 1 << 20, None) == -4
    assert L.hclsm_linear_attention_backward(block(_lib.HclsmLinearAttention, **{**base, "g": None}), P, 1 << 20, None) == -1
    assert L.hclsm_linear_attention_backward(block(_lib.HclsmLinearAttention, **{**base, "dq": P + 8}), P, 1 << 20, None) == -4
    long = {**base, "B": 1, "L": 1 << 16, "q_sb": 1 << 21, "k_sb": 1 << 21, "v_sb": 1 << 21, "g_sb": 1 << 21}
    for f in (L.hclsm_linear_attention_forward, L.hclsm_linear_attention_backward):     # workspace missing, short, unaligned
        assert f(block(_lib.HclsmLinearAttention, **long), None, 0, None) == -1
        assert f(block(_lib.HclsmLinearAttention, **long), P, 8, None) == -2
        assert f(block(_lib.HclsmLinearAttention, **long), P + 8, 1 << 40, None) == -4

    s = dict(q=P, k=P, v=P, log_decay=P, state=P, out=P, q_sb=32, q_sh=16, k_sb=32, k_sh=16, v_sb=32, v_sh=16, state_sb=512,
             n_states=2, B=2, H=2, Hk=2, dk=16, dv=16, scale=0.25, dtype=1)
    run = lambda **kw: L.hclsm_linear_attention_step(block(_lib.HclsmLinearAttentionStep, **{**s, **kw}), None)
    assert L.hclsm_linear_attention_step(None, None) == -1
    assert run(q=None) == -1 and run(state=None) == -1 and run(out=None) == -1
    assert run(n_states=1) == -2 and run(scale=0.0) == -2 and run(Hk=3) == -2
    assert run(dtype=5) == -3 and run(rows_dtype=2) == -3
    assert run(state=P + 4) == -4 and run(state_sb=510) == -4 and run(dv=12) == -4
    assert run(B=0) == 0


def test_blocks_are_packed_as_the_structs():
    from hclsm_amd import _lib
    for pack, fields, kind in ((_lib.pack_linear, _lib.LINEAR_FIELDS, _lib.HclsmLinearAttention),
                               (_lib.pack_step, _lib.STEP_FIELDS, _lib.HclsmLinearAttentionStep),
                               (_lib.pack_residual, _lib.RESIDUAL_FIELDS, _lib.HclsmResidualNorm)):
        names = sum(fields, ())
        raw = pack(*(i + 1 for i in range(len(names))))
        assert len(raw) == ctypes.sizeof(kind)
        b = kind.from_buffer_copy(raw)
        assert [int(getattr(b, n)) for n in names] == list(range(1, len(names) + 1))
