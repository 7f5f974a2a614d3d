"""torch.library ops of cross attention and of norms and rotations: empty sizes and refusals (argument checks on the CPU,
results on the GPU)."""

from __future__ import annotations

import pytest
import torch

import hclsm_amd.kernels.ops as ops

OPS = torch.ops.hclsm_hip

EMPTY = [(0, 3, 4, 2), (2, 0, 4, 2), (2, 3, 4, 0)]      # B, Lq, Lk, H: no batch row, no query, no query head


def _empty(B, Lq, Lk, H, dtype, device):
    q = torch.empty(B, Lq, H, 16, dtype=dtype, device=device)
    k, v = (torch.ones(B, Lk, 2, 16, dtype=dtype, device=device) for _ in range(2))
    return q, k, v, torch.empty(B, Lq, H, 16, dtype=dtype, device=device), torch.empty(B, H, Lq, device=device)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes", EMPTY)
def test_saved_outputs_of_empty_queries_pass_the_checks(sizes, dtype):
    q, _, _, out, lse = _empty(*sizes, dtype, "meta")
    for lo in (torch.empty(0, dtype=dtype, device="meta"), torch.empty_like(q)):
        assert ops._saved_lo(q, out, lse, lo) is None


def test_saved_outputs_of_other_shapes_are_refused():
    q, _, _, out, lse = _empty(2, 3, 4, 2, torch.bfloat16, "meta")
    lo = torch.empty_like(q)
    assert ops._saved_lo(q, out, lse, lo) is lo
    assert ops._saved_lo(q, out, lse, lo.new_empty(0)) is None
    for bad in ((out[:, :2], lse, lo), (out, lse[:1], lo), (out, lse, lo[:, :2]), (out.float(), lse, lo),
                (out, lse.double(), lo), (out, lse, lo.float())):
        with pytest.raises(ValueError, match="the forward's"):
            ops._saved_lo(q, *bad)


@pytest.mark.gpu
@pytest.mark.parametrize("for_grad", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes", EMPTY)
def test_empty_queries(sizes, dtype, for_grad):
    q, k, v, g, _ = _empty(*sizes, dtype, "cuda")
    out, lse, lo = OPS.cross_attention_fwd(q, k, v, None, None, None, 0.25, for_grad)
    dq, dk, dv = OPS.cross_attention_bwd(q, k, v, out, lse, lo, g, None, None, None, 0.25)
    assert (dq.shape, dk.shape, dv.shape) == (q.shape, k.shape, v.shape)
    assert not dk.any() and not dv.any()


def test_weights_without_a_norm_and_bad_eps_are_refused():
    w = torch.ones(16)
    ops._check_norm("f", w, 0.0, True)
    ops._check_norm("f", None, float("nan"), False)          # no norm: eps is not looked at
    with pytest.raises(ValueError, match="belongs to the norm"):
        ops._check_norm("f", w, 1e-6, False)
    for eps in (-1e-6, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            ops._check_norm("f", w, eps, True)


@pytest.mark.gpu
def test_norm_refusals_of_the_ops():
    x, w = torch.ones(1, 2, 3, 16, device="cuda"), torch.ones(16, device="cuda")
    with pytest.raises(ValueError, match="belongs to the norm"):
        OPS.norm_rotary_fwd(x, w, None, None, 0, 0, 1.0, 1e-6, False)
    with pytest.raises(ValueError, match="eps"):
        OPS.norm_rotary_fwd(x, w, None, None, 0, 0, 1.0, -1.0, True)
    with pytest.raises(ValueError, match="eps"):
        OPS.norm_rotary_bwd(x, w, None, None, x, 0, 0, 1.0, float("nan"))
