"""torch.library ops of cross attention and of norms and rotations: shapes on meta tensors and refusals (CPU), results
against the eager functions (GPU)."""

from __future__ import annotations

import pytest
import torch

import hclsm_amd.kernels.ops  # noqa: F401  (registers the ops)

OPS = torch.ops.hclsm_hip


def _m(*s, dt=torch.float32):
    return torch.empty(*s, device="meta", dtype=dt)


def test_fake_shapes():
    bf = torch.bfloat16
    q, k = _m(2, 5, 4, 16, dt=bf), _m(2, 9, 2, 16, dt=bf)
    out, lse, lo = OPS.cross_attention_fwd(q, k, k, None, None, None, 0.25, True)
    assert (out.shape, out.dtype, lse.shape, lse.dtype, lo.shape) == (q.shape, bf, (2, 4, 5), torch.float32, q.shape)
    assert OPS.cross_attention_fwd(q, k, k, None, None, None, 0.25, False)[2].shape == (0,)
    assert OPS.cross_attention_fwd(q.float(), k.float(), k.float(), None, None, None, 0.25, True)[2].shape == (0,)
    g = OPS.cross_attention_bwd(q, k, k, out, lse, lo, q, None, None, None, 0.25)
    assert [t.shape for t in g] == [q.shape, k.shape, k.shape]
    turns = _m(8, dt=torch.float64)
    assert OPS.norm_rotary_fwd(q, _m(16), turns, None, 16, 0, 1.0, 1e-6, True).shape == q.shape
    gx, gw = OPS.norm_rotary_bwd(q, _m(16), turns, None, q, 16, 0, 1.0, 1e-6)
    assert gx.shape == q.shape and (gw.shape, gw.dtype) == ((16,), torch.float32)
    assert OPS.norm_rotary_bwd(q, None, turns, None, q, 16, 0, 1.0, 1e-6)[1].shape == (0,)


def test_cpu_tensors_are_refused():
    x = torch.randn(1, 2, 3, 16)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        OPS.cross_attention_fwd(x, x, x, None, None, None, 0.25, False)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        OPS.norm_rotary_fwd(x, None, None, None, 0, 0, 1.0, 1e-6, True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ops_equal_eager(dtype):
    from hclsm_amd.kernels import RotaryPlan, cross_attention, qk_norm_rotary, rotary_embedding
    g = torch.Generator().manual_seed(3)
    q, go = (torch.randn(2, 40, 6, 64, generator=g).to(dtype).cuda() for _ in range(2))
    k, v = (torch.randn(2, 90, 2, 64, generator=g).to(dtype).cuda() for _ in range(2))
    lens = torch.tensor([90, 41], device="cuda")
    pad = torch.rand(2, 90, generator=g).cuda() < 0.2
    out, lse, lo = OPS.cross_attention_fwd(q, k, v, pad, lens, None, 0.125, True)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    eager, elog = cross_attention(*leaves, key_padding_mask=pad, key_lens=lens, scale=0.125, return_lse=True)
    assert torch.equal(out, eager) and torch.equal(lse, elog)
    grads = OPS.cross_attention_bwd(q, k, v, out, lse, lo, go, pad, lens, None, 0.125)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(eager, leaves, go)))
    with pytest.raises(ValueError):
        OPS.cross_attention_bwd(q, k, v, out[:, :3], lse, lo, go, pad, lens, None, 0.125)
    plan = RotaryPlan(32, layout="interleaved")
    turns = plan._turns[0].contiguous()
    w = (1 + 0.1 * torch.randn(64, generator=g)).cuda()
    y = OPS.norm_rotary_fwd(q, w, turns, lens[:1].expand(40), 32, 1, plan.amplitude, 1e-6, True)
    x, ww = q.clone().requires_grad_(), w.clone().requires_grad_()
    ye, _ = qk_norm_rotary(x, None, ww, None, plan, lens[:1].expand(40))
    assert torch.equal(y, ye)
    got = OPS.norm_rotary_bwd(q, w, turns, lens[:1].expand(40), go, 32, 1, plan.amplitude, 1e-6)
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(ye, (x, ww), go)))
    assert torch.equal(OPS.norm_rotary_fwd(q, None, turns, None, 32, 1, plan.amplitude, 0.0, False), rotary_embedding(q, plan))
    for bad in (dict(rot=33), dict(rot=66), dict(rot=34), dict(layout=2)):
        with pytest.raises(ValueError):
            OPS.norm_rotary_fwd(q, None, turns, None, bad.get("rot", 32), bad.get("layout", 1), 1.0, 0.0, False)
    checks = ("test_schema", "test_faketensor")
    torch.library.opcheck(OPS.cross_attention_fwd.default, (q, k, v, pad, lens, None, 0.125, True), test_utils=checks)
    torch.library.opcheck(OPS.norm_rotary_fwd.default, (q, w, turns, None, 32, 1, 1.0, 1e-6, True), test_utils=checks)
