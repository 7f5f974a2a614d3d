"""Sines and cosines of the rotation's angles against float64.

Of x in float32, |x| <= pi/4, and U = 2^-24: x is rounded once (U/2), and the last addition of either polynomial rounds its value (U/2
below one).  sin: 0.88 U/2 + U/2, and 2.6 U of the term x^3/6 and what follows, at most 0.09: 1.2 U.  cos: 0.71 U/2 + U/2, z = x^2
rounded (U z / 2 = 0.31 U) and the factor of z (U/4 of 0.62): 1.3 U.  Remainders of 2^-28 = 0.06 U.  Together at most 1.4 U."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_sines_and_cosines(layout):
    """The unit vector of every pair turned by 2^16 positions: (cos, sin) as they are."""
    from hclsm_amd.kernels import RotaryPlan, rotary_embedding
    n, L = 32, 1 << 16
    plan = RotaryPlan(2 * n, layout=layout)
    x = torch.zeros(1, L, 1, 2 * n, device="cuda")
    first, second = (slice(0, n), slice(n, None)) if layout == "half" else (slice(0, None, 2), slice(1, None, 2))
    x[..., first] = 1
    y = rotary_embedding(x, plan)[0, :, 0].double().cpu().numpy()
    angle = np.arange(L)[:, None] * plan.inv_freq.numpy()
    for got, ref in ((y[:, first], np.cos(angle)), (y[:, second], np.sin(angle))):
        err = np.abs(got - ref)
        print(f"{layout}: off by {err.max() * 2 ** 24:.2f} U, rms {np.sqrt((err ** 2).mean()) * 2 ** 24:.3f} U", flush=True)
        assert err.max() <= 1.4 * 2.0 ** -24
