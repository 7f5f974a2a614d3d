"""The residual norm on what is not finite, and on squares past float32."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_an_infinity_in_grouped_scales():
    """The mean of squares is infinite, and every other element of the row is zero times its weight; the infinity's own group is NaN."""
    from hclsm_amd.kernels import residual_rms_norm, residual_rms_norm_fp8
    x = torch.randn(3, 256, device="cuda")
    x[1, 70], x[2, 255] = float("inf"), float("-inf")
    y, s, _ = residual_rms_norm_fp8(x, group=64)
    for row, g in ((1, 1), (2, 3)):
        rest = [i for i in range(4) if i != g]
        assert torch.isnan(s[row, g]) and torch.isnan(y[row, 64 * g:64 * g + 64].float()).all()
        assert (s[row, rest] == 2.0 ** -100 / 448).all() and not y[row].float().view(4, 64)[rest].any()
        z = residual_rms_norm(x)[0][row]
        assert torch.isnan(z).sum() == 1 and not z.nan_to_num(0.0).any()
    assert torch.isfinite(y[0].float()).all()


def test_squares_past_float32():
    from hclsm_amd.kernels import residual_rms_norm, residual_rms_norm_fp8
    x = torch.full((2, 64), 1e20, device="cuda")
    x[1] = 1e18
    y, _ = residual_rms_norm(x)
    assert not y[0].any() and (y[1] - 1).abs().max() <= 48 * 2.0 ** -24      # (test_residual_norm_gpu.py)
    assert not residual_rms_norm_fp8(x, group=32)[0][0].float().any()
