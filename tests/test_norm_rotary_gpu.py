"""GPU parity of the norm and rotation of heads against oracle/heads.py (float64).

Tolerances, elementwise: half a step of the output type at the value (finfo.eps / 2), plus float32 arithmetic in units
of 2^-24 of the terms' size.  Forward: 12 for the root mean square (a sum of dh squares, at most 24 additions in
sequence, halved by the square root) + 2 for it and its product, 2 for the weight and the amplitude, 3.6 for the
angle (a turn rounded to float32 is off by 2^-26, times 2 pi) and its sine, 3 for the two products and their sum:
24 of |a| + |b| of the pair.  Backward: the rotation, the row's sum of products and the norm, each at most 24.
The weights' gradient adds up to 400 terms in sequence per element (at most 17 heads, 256 groups, 16 + 64 partial sums
here): 400 of the sum of the terms' magnitudes."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import heads as oh

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}   # half the subnormal step of fp16


def _np(t):
    return t.detach().double().cpu().numpy()


def _within(got, ref, scale, units, dtype, what):
    tol = torch.finfo(dtype).eps / 2 * np.abs(ref) + units * U * scale * (1 + torch.finfo(dtype).eps) + TINY[dtype]
    err = np.abs(_np(got) - ref)
    assert np.isfinite(_np(got)).all(), f"{what}: not finite"
    assert (err <= tol).all(), f"{what}: {(err - tol).max():.3e} over at {np.unravel_index((err - tol).argmax(), err.shape)}"


def _pair_scale(x, rot, layout):
    """|a| + |b| of an element's pair (|x| where it passes through)."""
    s = np.abs(x).copy()
    if rot:
        a, b = oh.pair_columns(rot, layout)
        s[..., a] = s[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return s


def _plan(rot, layout, **kw):
    from hclsm_amd.kernels import RotaryPlan
    return RotaryPlan(rot, layout=layout, **kw)


SHAPES = [  # B, L, H, dh, rot
    (1, 1, 1, 1, 0), (1, 1, 1, 2, 2), (3, 1, 12, 64, 64), (2, 7, 5, 64, 32), (1, 33, 3, 80, 40), (2, 5, 4, 80, 20),
    (1, 9, 13, 128, 126), (2, 3, 1, 256, 256), (1, 2, 9, 255, 2), (1, 4, 4, 33, 32), (2, 300, 6, 96, 96),
    (5, 3, 2, 64, 8), (1, 6, 4, 8, 4), (1, 5, 17, 192, 62),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_rotary_forward_and_backward(shape, layout, dtype):
    from hclsm_amd.kernels import qk_norm_rotary, rotary_embedding
    B, L, H, dh, rot = shape
    print(f"norm_rotary {shape} {layout} {dtype}", flush=True)
    g = torch.Generator().manual_seed(hash(shape) % 1000)
    Lk, Hk = max(1, L // 2), max(1, H // 2)
    q, gq = (torch.randn(B, L, H, dh, generator=g).to(dtype) for _ in range(2))
    k, gk = (3.0 * torch.randn(B, Lk, Hk, dh, generator=g).to(dtype) for _ in range(2))
    wq, wk = (1 + 0.3 * torch.randn(dh, generator=g) for _ in range(2))
    pos = torch.randint(0, 1 << 20, (B, L), generator=g)
    plan = _plan(rot, layout, scaling="yarn", factor=4.0, original_length=512) if rot else None
    freq, amp = (plan.inv_freq.numpy(), plan.amplitude) if rot else (None, 1.0)
    ins = [t.cuda().requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = qk_norm_rotary(*ins, plan, pos.cuda(), eps=1e-5)
    grads = torch.autograd.grad((yq, yk), ins, (gq.cuda(), gk.cuda()))
    for name, x, w, go, p, y, gx, gw in (("q", q, wq, gq, pos.numpy(), yq, grads[0], grads[2]),
                                         ("k", k, wk, gk, np.arange(Lk), yk, grads[1], grads[3])):
        x, w, go = _np(x), _np(w), _np(go)
        ref = oh.norm_rotate(x, w, p, freq, amp, layout, 1e-5)
        flat = oh.norm_rotate(x, w, p, None, eps=1e-5)
        _within(y, ref, amp * _pair_scale(flat, rot, layout), 24, dtype, name)
        rx, rw = oh.norm_rotate_grads(x, w, go, p, freq, amp, layout, 1e-5)
        r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5)
        n, d = np.abs(x * r), amp * _pair_scale(go, rot, layout)
        dn = d * np.abs(w)
        _within(gx, rx, r * (dn + n * (dn * n).mean(-1, keepdims=True)), 72, dtype, "d" + name)
        _within(gw, rw, (d * n).sum((0, 1, 2)), 400, torch.float32, "dw" + name)
    if rot:
        x = q.cuda().requires_grad_()
        y = rotary_embedding(x, plan, pos.cuda())
        (gx,) = torch.autograd.grad(y, x, gq.cuda())
        _within(y, oh.rotate(_np(q), pos, freq, amp, layout), amp * _pair_scale(_np(q), rot, layout), 10, dtype, "turned")
        _within(gx, oh.rotate(_np(gq), pos, freq, amp, layout, back=True), amp * _pair_scale(_np(gq), rot, layout), 10,
                dtype, "turned back")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_alignment_and_broadcast(dtype):
    """Views of a fused projection, rows at odd addresses, a batch repeated by stride 0, transposed heads."""
    from hclsm_amd.kernels import qk_norm_rotary, rotary_embedding
    g = torch.Generator().manual_seed(5)
    B, L, H, dh = 3, 10, 4, 64
    plan = _plan(64, "half")
    freq = plan.inv_freq.numpy()
    base = torch.randn(B, L, 3, H, dh, generator=g).to(dtype).cuda()
    odd = torch.randn(B, L, H, dh + 1, generator=g).to(dtype).cuda()
    views = {"fused": base[:, :, 1], "odd rows": odd[..., 1:], "stride 0": base[:1, :, 0].expand(B, L, H, dh),
             "heads first": base[:, :, 2].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3),
             "strided elements": torch.randn(B, L, H, 2 * dh, generator=g).to(dtype).cuda()[..., ::2]}
    for name, x in views.items():
        print(f"strides {name} {dtype}", flush=True)
        _within(rotary_embedding(x, plan), oh.rotate(_np(x), np.arange(L), freq),
                _pair_scale(_np(x), 64, "half"), 10, dtype, name)
    w = torch.ones(dh, device="cuda")
    x = base.clone().requires_grad_()
    y, _ = qk_norm_rotary(x[:, :, 1], None, w, None, plan)
    (gx,) = torch.autograd.grad(y.sum(), x)                       # a gradient of stride 0
    rx, _ = oh.norm_rotate_grads(_np(base[:, :, 1]), np.ones(dh), np.ones((B, L, H, dh)), np.arange(L), freq)
    r = 1 / np.sqrt((_np(base[:, :, 1]) ** 2).mean(-1, keepdims=True))
    n = np.abs(_np(base[:, :, 1])) * r
    _within(gx[:, :, 1], rx, r * (2 + n * 2 * n.mean(-1, keepdims=True)), 72, dtype, "gradient of a view")
    assert not gx[:, :, 0].any() and not gx[:, :, 2].any()


def test_far_and_negative_positions_and_types():
    """Positions to 2^31 and below zero keep float32 angles; int32, int64, (L,) and (B, L) agree bit for bit."""
    from hclsm_amd.kernels import rotary_embedding
    g = torch.Generator().manual_seed(6)
    pos = torch.tensor([0, -5, 1 << 20, (1 << 31) - 1, -(1 << 31) + 1, 12345])
    x = torch.randn(2, 6, 3, 32, generator=g)
    plan = _plan(32, "interleaved")
    y = rotary_embedding(x.cuda(), plan, pos.cuda())
    # 2^31 turns of float64 leave 2^-22 of a turn in either computation: 2 * 2 pi * 4 units
    _within(y, oh.rotate(_np(x), pos, plan.inv_freq.numpy(), 1.0, "interleaved"), _pair_scale(_np(x), 32, "interleaved"),
            10 + 52, torch.float32, "far")
    for p in (pos.int(), pos.expand(2, 6), pos.int().expand(2, 6).contiguous(), torch.stack((pos, pos), 1)[:, 0]):
        assert torch.equal(rotary_embedding(x.cuda(), plan, p.cuda()), y)


def test_gradients_against_differences():
    """<gradient, direction> of the float32 kernels against central differences of the float64 statement."""
    from hclsm_amd.kernels import qk_norm_rotary
    r = np.random.default_rng(7)
    x, w, go = r.normal(size=(2, 9, 3, 48)), 1 + 0.2 * r.normal(size=48), r.normal(size=(2, 9, 3, 48))
    plan = _plan(36, "half", scaling="linear", factor=2.0)
    f32 = lambda t: torch.tensor(t, dtype=torch.float32).cuda()
    x, w, go = (np.float64(np.float32(t)) for t in (x, w, go))
    tx, tw = f32(x).requires_grad_(), f32(w).requires_grad_()
    y, _ = qk_norm_rotary(tx, None, tw, None, plan, eps=1e-6)
    gx, gw = torch.autograd.grad(y, (tx, tw), f32(go))
    f = lambda x, w: (go * oh.norm_rotate(x, w, np.arange(9), plan.inv_freq.numpy())).sum()
    h = 1e-5
    ux, uw = r.normal(size=x.shape), r.normal(size=48)
    for got, u, diff in ((gx, ux, f(x + h * ux, w) - f(x - h * ux, w)), (gw, uw, f(x, w + h * uw) - f(x, w - h * uw))):
        terms = np.abs(_np(got) * u).sum()
        assert abs((_np(got) * u).sum() - diff / (2 * h)) <= 500 * U * terms + 1e-7 * terms


def test_empty_tensors_and_special_rows():
    from hclsm_amd.kernels import qk_norm_rotary, rotary_embedding
    plan = _plan(16, "half")
    for shape in ((0, 4, 2, 16), (2, 0, 2, 16), (2, 4, 0, 16)):
        assert rotary_embedding(torch.empty(shape, device="cuda"), plan).shape == shape
        q = torch.empty(shape, device="cuda", requires_grad=True)
        w = torch.ones(16, device="cuda", requires_grad=True)
        k = torch.randn(1, 2, 3, 16, device="cuda", requires_grad=True)
        yq, yk = qk_norm_rotary(q, k, w, w, plan)
        gq, gk, gw = torch.autograd.grad((yq, yk), (q, k, w), (torch.ones_like(yq), torch.ones_like(yk)))
        assert gq.shape == shape and torch.isfinite(gk).all()
        ref = oh.norm_rotate_grads(_np(k), np.ones(16), np.ones(k.shape), np.arange(2), plan.inv_freq.numpy())[1]
        np.testing.assert_allclose(_np(gw), ref, atol=400 * U * 64)
    # a zero row is scaled by 1/sqrt(eps); a row with a NaN leaves its neighbours alone
    x = torch.randn(1, 3, 2, 16)
    x[0, 1, 0] = 0
    x[0, 2, 1, 5] = float("nan")
    y, _ = qk_norm_rotary(x.cuda(), None, None, None, plan)
    y = y.cpu()
    assert not y[0, 1, 0].any() and y[0, 2, 1].isnan().all() and torch.isfinite(y[0, 2, 0]).all()
    assert torch.isfinite(y[0, :2]).all()


def test_weights_dtypes_and_partial_gradients():
    """Weights in the heads' type, gradients of some inputs only, twice the same result (no atomics)."""
    from hclsm_amd.kernels import qk_norm_rotary
    g = torch.Generator().manual_seed(9)
    q, k = (torch.randn(4, 33, 6, 64, generator=g).bfloat16().cuda() for _ in range(2))
    w = (1 + 0.1 * torch.randn(64, generator=g)).bfloat16().cuda().requires_grad_()
    plan = _plan(64, "half")
    y, _ = qk_norm_rotary(q, k, w, None, plan)
    go = torch.randn(y.shape, generator=g).bfloat16().cuda()
    (gw,) = torch.autograd.grad(y, w, go, retain_graph=True)
    _, rw = oh.norm_rotate_grads(_np(q), _np(w), _np(go), np.arange(33), plan.inv_freq.numpy())
    n = np.abs(_np(q)) / np.sqrt((_np(q) ** 2).mean(-1, keepdims=True))
    _within(gw, rw, (_pair_scale(_np(go), 64, "half") * n).sum((0, 1, 2)), 400, torch.bfloat16, "dw")
    assert gw.dtype == torch.bfloat16 and torch.equal(gw, torch.autograd.grad(y, w, go)[0])


def test_graph_replays_and_side_stream():
    from hclsm_amd.kernels import qk_norm_rotary
    g = torch.Generator().manual_seed(10)
    q, k = torch.randn(8, 1, 12, 64, generator=g).bfloat16().cuda(), torch.randn(8, 1, 4, 64, generator=g).bfloat16().cuda()
    w = torch.ones(64, device="cuda")
    pos = torch.arange(8, device="cuda")[:, None] * 1000
    plan = _plan(64, "half")
    qk_norm_rotary(q, k, w, w, plan, pos, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yq, yk = qk_norm_rotary(q, k, w, w, plan, pos, pos)
    side = torch.cuda.Stream()
    for step in range(3):
        q.normal_(generator=torch.Generator("cuda").manual_seed(step))
        pos.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        ref = qk_norm_rotary(q, k, w, w, plan, pos, pos)
        assert torch.equal(yq, ref[0]) and torch.equal(yk, ref[1])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = qk_norm_rotary(q, k, w, w, plan, pos, pos)
        side.synchronize()
        assert torch.equal(other[0], ref[0])
    del graph
