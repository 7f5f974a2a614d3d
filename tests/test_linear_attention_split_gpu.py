"""Linear attention's ways through its launches: the same bits whichever gradients are asked for."""

from __future__ import annotations

import pytest
import torch

from test_linear_attention_gpu import BF16, F16, F32, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dk,dv", [(F16, 64, 128), (BF16, 64, 256), (F32, 128, 48), (F16, 256, 64), (BF16, 128, 64)])
@pytest.mark.parametrize("B", [2, 200])
def test_any_gradient_alone_has_the_bits_it_has_with_all(dtype, dk, dv, B):
    from hclsm_amd.kernels import linear_attention
    q, k, v, s0, decay, go, gs = (t.cuda() for t in _inputs(B, 150, 2, 1, dk, dv, dtype, 33))

    def grads(need):
        t = [x.clone().requires_grad_(n) for x, n in zip((q, k, v, s0), need)]
        o = linear_attention(*t[:3], decay, initial_state=t[3], return_state=True)
        return torch.autograd.grad(o, [x for x in t if x.requires_grad], (go, gs))
    full = grads([True] * 4)
    for need in ([0], [1], [2], [3], [0, 1], [2, 3], [1, 2]):
        for i, got in zip(need, grads([j in need for j in range(4)])):
            assert torch.equal(got, full[i]), (need, i)
