"""16-bit forwards of 17 to 32 rows of a key head (a frame's slots) with heads up to 64: the weights in two operands, so that
the output is off by little more than its own rounding (bounds in cross_attention_bounds.py, fine)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cross_attention_bounds import assert_within, bounds
from oracle import heads as oh

pytestmark = pytest.mark.gpu

SHAPES = [(2, 32, 196, 3, 3, 64), (1, 3, 400, 8, 1, 40), (2, 17, 1003, 2, 2, 32), (1, 1, 5000, 20, 1, 64), (3, 31, 33, 2, 2, 8),
          (700, 20, 70, 1, 1, 48)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_outputs_of_up_to_32_rows(shape, masked, dtype):
    from hclsm_amd.kernels import cross_attention
    B, Lq, Lk, H, Hk, dh = shape
    print(f"{shape} {dtype} masked {masked}", flush=True)
    gen = torch.Generator().manual_seed(51)
    q, k, v = (torch.randn(B, L, h, dh, generator=gen).to(dtype) for L, h in ((Lq, H), (Lk, Hk), (Lk, Hk)))
    live, masks = np.ones((B, Lk), bool), {}
    if masked:
        lens = torch.randint(0, Lk + 1, (B,), generator=gen)
        pad = torch.rand(B, Lk, generator=gen) < 0.2
        live = (np.arange(Lk) < lens.numpy()[:, None]) & ~pad.numpy()
        v[torch.tensor(~live)] = float("nan")
        masks = dict(key_lens=lens.cuda(), key_padding_mask=pad.cuda())
    with torch.no_grad():
        got = cross_attention(q.cuda(), k.cuda(), v.cuda(), **masks)
    vals = [t.double().numpy() for t in (q, k, v)]
    vals[2] = np.where(live[:, :, None, None], vals[2], 0)
    ref, _ = oh.cross_attention(*vals, live)
    assert_within(got, ref, bounds(*vals, live, None, None, dtype, fine=True)[0], f"{shape} {dtype}")
