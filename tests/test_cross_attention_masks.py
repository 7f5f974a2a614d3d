"""key_padding_mask of other types than bool (CPU: the mask as the kernels read it)."""

from __future__ import annotations

import importlib
import warnings

import pytest
import torch


def _mask(pad):
    return importlib.import_module("hclsm_amd.kernels.cross_attention")._masks(pad, None, None)[0]


FLAGS = torch.tensor([[True, False, True], [False, False, True]])


@pytest.mark.parametrize("dtype", [torch.bool, torch.uint8, torch.int32, torch.int64])
def test_flags(dtype):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        got = _mask(FLAGS.to(dtype))
    assert got.dtype in (torch.bool, torch.uint8) and torch.equal(got.bool(), FLAGS)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_float_masks_are_flags_and_say_so(dtype):
    """Also a finite entry, which nn.MultiheadAttention would add to the scores."""
    pad = torch.tensor([[float("-inf"), 0.0, -2.5], [-0.0, 0.0, 1.0]], dtype=dtype)
    with pytest.warns(UserWarning, match="read as flags"):
        got = _mask(pad)
    assert torch.equal(got, FLAGS)
