"""torch.library ops of linear attention and of norms with the residual: shapes on meta tensors and refusals (CPU), results
against the eager functions (GPU)."""

from __future__ import annotations

import pytest
import torch

import hclsm_amd.kernels.ops  # noqa: F401  (registers the ops)

OPS = torch.ops.hclsm_hip
BF = torch.bfloat16


def _m(*s, dt=torch.float32):
    return torch.empty(*s, device="meta", dtype=dt)


def test_fake_shapes():
    q, k, v, s = _m(2, 5, 4, 16, dt=BF), _m(2, 5, 2, 16, dt=BF), _m(2, 5, 2, 24, dt=BF), _m(2, 4, 16, 24)
    d = _m(4)
    out, s1 = OPS.linear_attention_fwd(q, k, v, d, None, None, 0.25, True)
    assert (out.shape, out.dtype, s1.shape, s1.dtype) == ((2, 5, 4, 24), BF, s.shape, torch.float32)
    assert OPS.linear_attention_fwd(q, k, v, d, s, None, 0.25, False)[1].shape == (0,)
    g = OPS.linear_attention_bwd(q, k, v, d, s, None, out, s, 0.25)
    assert [t.shape for t in g] == [q.shape, k.shape, v.shape, s.shape] and g[3].dtype == torch.float32
    assert OPS.linear_attention_bwd(q, k, v, d, None, None, out, None, 0.25)[3].shape == (0,)
    assert OPS.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], d, s, None, 0.25).shape == (2, 4, 24)
    x, r, w = _m(3, 7, 64, dt=BF), _m(3, 7, 64), _m(64)
    y, h = OPS.residual_rms_norm_fwd(x, r, w, 1e-6)
    assert (y.shape, y.dtype, h.shape, h.dtype) == (x.shape, BF, x.shape, torch.float32)
    assert OPS.residual_rms_norm_fwd(x, None, w, 1e-6)[1].shape == (0,)
    y8, sc, h = OPS.residual_rms_norm_fp8(x, r, w, 1e-6, 32)
    assert (y8.dtype, sc.shape, h.dtype) == (torch.float8_e4m3fn, (3, 7, 2), torch.float32)
    assert OPS.residual_rms_norm_fp8(x, None, w, 1e-6, 0)[1].shape == (3, 7, 1)
    dx, dr, dw = OPS.residual_rms_norm_bwd(r, w, x, r, 1e-6)
    assert (dx.dtype, dr.dtype, dw.shape) == (BF, torch.float32, (64,))
    dx, dr, dw = OPS.residual_rms_norm_bwd(x, None, x, None, 1e-6)
    assert dr.shape == (0,) and dw.shape == (0,)


def test_cpu_tensors_are_refused():
    x, d = torch.randn(1, 2, 3, 16), torch.zeros(3)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        OPS.linear_attention_fwd(x, x, x, d, None, None, 0.25, False)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        OPS.linear_attention_step(x[:, 0], x[:, 0], x[:, 0], d, torch.zeros(1, 3, 16, 16), None, 0.25)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        OPS.residual_rms_norm_fwd(x, None, None, 1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_ops_equal_eager(dtype):
    from hclsm_amd.kernels import linear_attention, linear_attention_step, residual_rms_norm, residual_rms_norm_fp8
    g = torch.Generator().manual_seed(3)
    r = lambda *s, dt=dtype: torch.randn(*s, generator=g).to(dt).cuda()
    q, k, v, go = r(2, 90, 4, 32), r(2, 90, 2, 32), r(2, 90, 2, 64), r(2, 90, 4, 64)
    s, gs = r(2, 4, 32, 64, dt=torch.float32), r(2, 4, 32, 64, dt=torch.float32)
    d, lens = -torch.rand(4, generator=g).cuda(), torch.tensor([90, 41], device="cuda")
    got = OPS.linear_attention_fwd(q, k, v, d, s, lens, 0.2, True)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, s)]
    eager = linear_attention(*leaves[:3], d, initial_state=leaves[3], seq_lens=lens, scale=0.2, return_state=True)
    assert all(torch.equal(a, b) for a, b in zip(got, eager))
    grads = OPS.linear_attention_bwd(q, k, v, d, s, lens, go, gs, 0.2)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(eager, leaves, (go, gs))))
    with pytest.raises(ValueError):
        OPS.linear_attention_bwd(q, k, v, d, s, lens, go[:, :3], gs, 0.2)
    one, two = s.clone(), s.clone()
    rows = torch.tensor([1, 0], device="cuda")
    y = OPS.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], d, one, rows, 0.2)
    assert torch.equal(y, linear_attention_step(q[:, 0], k[:, 0], v[:, 0], d, two, rows=rows, scale=0.2))
    assert torch.equal(one, two)
    x, res, w, gy = r(33, 96), r(33, 96, dt=torch.float32), r(96, dt=torch.float32), r(33, 96)
    ins = [t.clone().requires_grad_() for t in (x, res, w)]
    y, h = residual_rms_norm(*ins)
    assert all(torch.equal(a, b) for a, b in zip(OPS.residual_rms_norm_fwd(x, res, w, 1e-6), (y, h)))
    want = torch.autograd.grad((y, h), ins, (gy, res))
    dx, dr, dw = OPS.residual_rms_norm_bwd(h.detach(), w, gy, res, 1e-6)
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[2]) and torch.equal(dr if dr.numel() else dx, want[1])
    for a, b in zip(OPS.residual_rms_norm_fp8(x, res, w, 1e-6, 32), residual_rms_norm_fp8(x, res, w, group=32)):
        assert torch.equal(a.float(), b.float())
    with pytest.raises(ValueError):
        OPS.residual_rms_norm_fp8(x, res, w, 1e-6, 48)
    checks = ("test_schema", "test_faketensor")
    torch.library.opcheck(OPS.linear_attention_fwd.default, (q, k, v, d, s, lens, 0.2, True), test_utils=checks)
    torch.library.opcheck(OPS.linear_attention_step.default, (q[:, 0], k[:, 0], v[:, 0], d, one, rows, 0.2), test_utils=checks)
    torch.library.opcheck(OPS.residual_rms_norm_fwd.default, (x, res, w, 1e-6), test_utils=checks)
