"""cross_attention of tensors whose rows are not where the kernels read them: what is copied (CPU) and results (GPU)."""

from __future__ import annotations

import importlib

import pytest
import torch

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _off(t, elements=1):
    """A contiguous tensor of t's values whose address is `elements` past a 16-byte boundary."""
    flat = torch.empty(t.numel() + 16, dtype=t.dtype, device=t.device)
    first = -flat.data_ptr() % 16 // t.element_size() + elements
    x = flat[first:first + t.numel()].view(t.shape)
    x.copy_(t)
    return x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2, 3, 4, 64), (1, 3, 4, 64), (2, 1, 1, 8)])
def test_contiguous_rows_off_a_boundary_are_copied(shape, dtype):
    rows = importlib.import_module("hclsm_amd.kernels.cross_attention")._rows
    t = torch.randn(shape).to(dtype)
    for elements in (1, 16 // t.element_size() - 1):
        x = _off(t, elements)
        assert x.is_contiguous() and x.data_ptr() % 16 == elements * t.element_size()
        y = rows(x)
        assert y.data_ptr() % 16 == 0 and y.is_contiguous() and torch.equal(y, t)
    on = _off(t, 0)
    assert rows(on) is on


@pytest.mark.parametrize("dtype", DTYPES)
def test_other_strides_are_copied_or_read_as_they_stand(dtype):
    rows = importlib.import_module("hclsm_amd.kernels.cross_attention")._rows
    t = torch.randn(2, 3, 4, 64).to(dtype)
    for x in (torch.cat((t[..., :1], t), -1)[..., 1:], torch.stack((t, t), -1).flatten(-2)[..., ::2],
              _off(t.permute(0, 2, 1, 3).contiguous()).permute(0, 2, 1, 3), t[..., :1].expand(2, 3, 4, 64)):
        y = rows(x)
        assert y.data_ptr() % 16 == 0 and y.is_contiguous() and torch.equal(y, x)
    for x in (t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), t[:1].expand(5, 3, 4, 64), t[:, :1].expand(2, 9, 4, 64),
              torch.stack((t, t), 2)[:, :, 1]):
        if x.data_ptr() % 16 == 0:
            assert rows(x) is x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Lq", [3, 70])
def test_contiguous_tensors_off_a_boundary(Lq, dtype):
    """q, k, v and the gradient as slices of flat buffers, each alone and all together: the same bits as aligned ones."""
    from hclsm_amd.kernels import cross_attention
    gen = torch.Generator().manual_seed(31)
    ts = [torch.randn(s, generator=gen).to(dtype).cuda() for s in ((2, Lq, 4, 64), (2, 90, 2, 64), (2, 90, 2, 64), (2, Lq, 4, 64))]

    def step(q, k, v, g):
        ins = [t.detach().requires_grad_() for t in (q, k, v)]
        out = cross_attention(*ins)
        return (out.detach(), *torch.autograd.grad(out, ins, g))

    ref = step(*ts)
    for which in ((0,), (1,), (2,), (3,), (0, 1, 2, 3)):
        moved = [_off(t) if i in which else t for i, t in enumerate(ts)]
        assert all(torch.equal(a, b) for a, b in zip(step(*moved), ref)), which


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_caches_with_heads_first_are_read_as_they_stand(dtype):
    """Heads of keys far apart, (B, H, L, dh) in memory, and tokens far apart, (L, B, H, dh): no copy.  (Nothing is touched here.)"""
    rows = importlib.import_module("hclsm_amd.kernels.cross_attention")._rows
    heads = torch.empty(1, 4, 1 << 20, 64, dtype=dtype).permute(0, 2, 1, 3)
    assert heads.stride(2) * 4 == 1 << 28 and rows(heads, True) is heads
    tokens = torch.empty(64, 1 << 21, dtype=dtype).as_strided((2, 60, 2, 64), (128, 1 << 21, 64, 1))
    assert rows(tokens, True) is tokens
    near = tokens[:, :1]
    assert rows(near) is near


@pytest.mark.gpu
@pytest.mark.parametrize("Lq", [2, 70])
def test_long_caches_with_heads_first(Lq):
    """The same bits from a cache with 2^27 elements between heads, or 2^21 between tokens, as from a compact one."""
    from hclsm_amd.kernels import cross_attention
    gen = torch.Generator().manual_seed(32)
    q, g = (torch.randn(1, Lq, 4, 64, generator=gen).bfloat16().cuda() for _ in range(2))
    k, v = (torch.randn(1, 150, 4, 64, generator=gen).bfloat16().cuda() for _ in range(2))
    far = torch.zeros(1, 4, 1 << 21, 64, dtype=torch.bfloat16, device="cuda").permute(0, 2, 1, 3)[:, :150]
    apart = torch.zeros(150, 1 << 21, dtype=torch.bfloat16, device="cuda").as_strided((1, 150, 4, 64), (256, 1 << 21, 64, 1))
    far.copy_(k), apart.copy_(v)

    def step(k, v):
        ins = [t.detach().requires_grad_() for t in (q, k, v)]
        out = cross_attention(*ins)
        return (out.detach(), *torch.autograd.grad(out, ins, g))

    assert far.stride(2) == 1 << 27
    assert all(torch.equal(a, b) for a, b in zip(step(far, apart), step(k, v)))
