"""Linear attention's ways through its launches: many segments of a long stream, jobs of different padded sizes with and without
a launch in common, and the same bits whichever gradients are asked for.  Tolerances: test_linear_attention_gpu.py."""

from __future__ import annotations

import pytest
import torch

from test_linear_attention_gpu import BF16, F16, F32, _compare, _inputs

pytestmark = pytest.mark.gpu

CODE = {F32: 0, BF16: 1, F16: 2}


def _segments(B, L, H, dk, dv, dtype, backward):
    from hclsm_amd import _lib
    n = _lib.lib().hclsm_linear_attention_workspace(B, L, H, H, dk, dv, CODE[dtype], backward)
    return n // ((3 if backward else 1) * B * H * dk * dv * 4)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("state", [False, True])
def test_more_than_32_segments(dtype, state):
    """Segments' states by a launch of their own, more than two of its rounds of 16; lengths inside a segment, on its border, one
    token either side of it, and none."""
    B, L, H, dk, dv = 2, 8700, 2, 32, 24
    chunks = -(-L // (32 if dtype == F32 else 64))
    n = [_segments(B, L, H, dk, dv, dtype, bwd) for bwd in (0, 1)]
    assert min(n) > 32, n
    border = 20 * -(-chunks // n[0]) * (32 if dtype == F32 else 64)
    ins = list(_inputs(B, L, H, H, dk, dv, dtype, 31, state))
    ins[4] = torch.tensor([-1e-3, -0.05])
    for lens in (None, [border, border + 1], [border - 1, 5000], [0, 8699]):
        print(f"{n} segments, {dtype}, {lens}", flush=True)
        _compare(*ins, lens=lens)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(130, 70, 1, 1, 64, 128), (45, 70, 2, 1, 48, 256), (66, 37, 2, 2, 136, 64)])
def test_a_launch_for_each_padded_size(shape, dtype):
    """More workgroups than are on the chip at once: jobs of dk and of dv padded differently run one after the other."""
    B, L, H, Hk, dk, dv = shape
    tiles = lambda d: -(-d // 64)
    assert B * H * (tiles(dv) + 2 * tiles(dk)) > 512 and _segments(B, L, H, dk, dv, dtype, 1) == 0
    print(f"launches {shape} {dtype}", flush=True)
    _compare(*_inputs(*shape, dtype, 32))


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
