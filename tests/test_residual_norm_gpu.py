"""GPU parity of the residual norm against oracle/residual_norm.py (float64), elementwise.

The stream is the sum rounded once, bit for bit.  Tolerances: half a step of the output type at the value (finfo.eps / 2), plus
float32 arithmetic in units of 2^-24 of the terms' sizes.  Forward: the mean of squares is a sum of at most 64 products in a
thread and 16 more additions over threads, halved by the root, 3 for root and mean, 2 products: 48.  Backward: the same sums in
both factors and four more operations: 120 of i (|gy w| + |n| mean(|gy w n|)) + |gh|.  The weight's gradient adds at most
rows / 1024 + 3 terms in a thread and group and 16 + 64 partial sums, each with the error of n (52): 160 + rows / 1024 here.
8 bits: half a step of e4m3 (2^-4 of the value, 2^-10 below 2^-6) of y / scale, whose own error is that of y and two roundings;
a value that close to the middle of two may go to either."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import residual_norm as on

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TINY = {F32: 0.0, BF16: 0.0, F16: 2.0 ** -25}


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _within(got, ref, M, units, what):
    got_, dt = _np(got), got.dtype
    tol = torch.finfo(dt).eps / 2 * np.abs(ref) + units * U * M * (1 + torch.finfo(dt).eps) + TINY[dt]
    assert got_.shape == ref.shape and np.isfinite(got_).all(), what
    err = np.abs(got_ - ref)
    assert (err <= tol).all(), f"{what}: {(err - tol).max():.3e} over at {np.unravel_index((err - tol).argmax(), err.shape)}"


def _inputs(shape, dtype, stream, wdt, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, gy = (torch.randn(*shape, generator=g).to(dtype).cuda() for _ in range(2))
    r = None if stream is None else (3 * torch.randn(*shape, generator=g)).to(stream).cuda()
    w = None if wdt is None else (1 + 0.3 * torch.randn(shape[-1], generator=g)).to(wdt).cuda()
    gh = torch.randn(*shape, generator=g).to(stream or dtype).cuda()
    return x, r, w, gy, gh


def _compare(x, r, w, gy, gh, eps):
    from hclsm_amd.kernels import residual_rms_norm
    ins = [None if t is None else t.detach().requires_grad_() for t in (x, r, w)]
    y, h = residual_rms_norm(*ins, eps=eps)
    if r is None:
        assert h.data_ptr() == ins[0].data_ptr() and h.shape == x.shape
    else:
        assert h.dtype == r.dtype and torch.equal(h, (x.float() + r.float()).to(r.dtype))
    hn, wn = _np(h), _np(w)
    ref = on.rms_norm(hn, wn, eps)
    _within(y, ref, np.abs(ref), 48, "y")
    assert y.dtype == x.dtype
    leaves = [t for t in ins if t is not None]
    got = list(torch.autograd.grad((y, h), leaves, (gy, gh)))
    dh, dw = on.rms_norm_grads(hn, _np(gy), _np(gh), wn, eps)
    i = 1 / np.sqrt((hn * hn).mean(-1, keepdims=True) + eps)
    n, gw = np.abs(hn * i), np.abs(_np(gy) * (1 if wn is None else wn))
    M = i * (gw + n * (gw * n).mean(-1, keepdims=True)) + np.abs(_np(gh))
    _within(got[0], dh, M, 120, "dx")
    if r is not None:
        _within(got[1], dh, M, 120, "dr")
        assert got[1].dtype == r.dtype
    assert got[0].dtype == x.dtype
    if w is not None:
        D = x.shape[-1]
        mag = (np.abs(_np(gy)) * n).reshape(-1, D).sum(0)
        _within(got[-1], dw, mag, 160 + x.numel() // D / 1024, "dw")


SHAPES = [(1, 1), (3, 7), (2, 5, 8), (5, 64), (1, 384), (9, 512), (33, 513), (4, 768), (7, 1000), (3, 1001), (2, 1536), (5, 2048),
          (2, 4096), (3, 4100), (2, 5001), (2, 8192), (1, 16384), (2, 16383), (2050, 40), (1100, 260)]


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32), (BF16, None), (F32, None)])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(shape, types):
    print(f"residual norm {shape} {types}", flush=True)
    wdt = {0: None, 1: F32, 2: types[0]}[shape[-1] % 3]
    _compare(*_inputs(shape, types[0], types[1], wdt), eps=1e-5)


def _check_fp8(x, r, w, group, eps=1e-6):
    from hclsm_amd.kernels import residual_rms_norm, residual_rms_norm_fp8
    y8, scale, h = residual_rms_norm_fp8(x, r, w, eps=eps, group=group)
    D = x.shape[-1]
    assert y8.dtype == torch.float8_e4m3fn and y8.shape == x.shape and scale.dtype == F32
    assert scale.shape == (*x.shape[:-1], D // group if group else 1)
    y, h2 = residual_rms_norm(x, r, w, eps=eps)
    assert torch.equal(h, h2)
    ref = on.rms_norm(_np(h), _np(w), eps)
    want = on.scales(ref, group or 0)
    assert (np.abs(_np(scale) - want) <= 50 * U * want).all()
    got = y8.cpu().float().double().numpy()
    t = (ref.reshape(*want.shape, -1) / want[..., None]).reshape(ref.shape)
    assert np.isfinite(got).all()
    assert (np.abs(got - t) <= np.maximum(np.abs(t) * 2.0 ** -4, 2.0 ** -10) + 110 * U * np.abs(t)).all()
    top = np.abs(got.reshape(*want.shape, -1)).max(-1)
    assert ((top == 448) | (want <= 2.0 ** -100 / 448)).all()       # the largest of a group has the largest value


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F16, F32), (BF16, None)])
@pytest.mark.parametrize("case", [((1, 1), None), ((3, 7), None), ((5, 384), None), ((4, 768), 128), ((3, 1001), None),
                                  ((2, 3, 4096), 32), ((9, 96), 32), ((2, 1600), 64), ((2, 8192), 128), ((2, 5000), None),
                                  ((1, 16384), 64), ((700, 32), 32), ((3, 2048), None)])
def test_eight_bits(case, types):
    shape, group = case
    print(f"8 bits {shape} {group} {types}", flush=True)
    x, r, w, _, _ = _inputs(shape, *types, F32, 3)
    _check_fp8(x, r, w, group)


def test_eight_bits_of_zeros_and_of_what_is_not_finite():
    from hclsm_amd.kernels import residual_rms_norm_fp8
    x = torch.randn(4, 128, device="cuda")
    x[0] = 0
    x[1, :64] = 0
    x[2, 3] = float("nan")
    x[3, 5] = float("inf")
    y, s, _ = residual_rms_norm_fp8(x, group=32)
    assert not y[0].float().any() and (s[0] == 2.0 ** -100 / 448).all() and (s[1, :2] == 2.0 ** -100 / 448).all()
    assert s[1, 2:].gt(1e-4).all() and not y[1, :64].float().any()
    assert torch.isnan(y[2].float()).all() and torch.isnan(s[2]).all()
    assert torch.isnan(s[3, 0]) and torch.isnan(y[3, :32].float()).all()
    y, s, _ = residual_rms_norm_fp8(x)
    assert not y[0].float().any() and torch.isnan(s[2:]).all() and torch.isnan(y[2:].float()).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_alignment(dtype):
    """Rows of a wider matrix, rows at odd addresses, a row repeated, transposed and strided views, higher dimensions."""
    from hclsm_amd.kernels import residual_rms_norm
    g = torch.Generator().manual_seed(5)
    base = torch.randn(12, 512, generator=g).to(dtype).cuda()
    w = (1 + 0.1 * torch.randn(2 * 256, generator=g)).cuda()[::2]
    views = {"wide": base[:, 256:], "odd": base[:, 1:257], "repeated": base[:1, :256].expand(12, 256), "every other row": base[::2, :256],
             "strided": base[:, ::2], "transposed": base.t().contiguous().t()[:, :256], "three": base.view(3, 4, 512)[:, 1:, :256],
             "vector": base[0, :256]}
    for name, x in views.items():
        print(f"strides {name} {dtype}", flush=True)
        r = base.flip(0).contiguous()[: x.shape[0], :256].expand_as(x) if x.dim() == 2 else x
        gy, gh = torch.ones(1, device="cuda").to(dtype).expand(x.shape), x
        _compare(x, r, w.contiguous(), gy, gh, 1e-6)
        assert torch.equal(residual_rms_norm(x, r, w)[0], residual_rms_norm(x, r, w.contiguous())[0])     # a strided weight
        if x.dim() == 2:
            _check_fp8(x, r, w, 32)
            _check_fp8(x, r, w, None)


def test_some_gradients_alone_and_none():
    from hclsm_amd.kernels import residual_rms_norm
    x, r, w, gy, gh = _inputs((40, 96), BF16, F32, F32, 6)

    def run(need, outs=(True, True)):
        leaf = [t.clone().requires_grad_(n) for t, n in zip((x, r, w), need)]
        ys = [o for o, u in zip(residual_rms_norm(*leaf), outs) if u]
        return torch.autograd.grad(ys, [t for t in leaf if t.requires_grad], [g for g, u in zip((gy, gh), outs) if u],
                                   allow_unused=True)
    full = run((True, True, True))
    for i in range(3):
        assert torch.equal(run([j == i for j in range(3)])[0], full[i])
    dx, dr, dw = run((True, True, True), (False, True))
    assert torch.equal(dr, gh) and torch.equal(dx, gh.to(BF16)) and not dw.any()
    empty = torch.empty(0, 96, device="cuda", requires_grad=True)
    ww = torch.ones(96, device="cuda", requires_grad=True)
    y, h = residual_rms_norm(empty, empty, ww)
    assert y.shape == (0, 96)
    assert not torch.autograd.grad(y.sum(), ww)[0].any()


def test_gradients_against_differences():
    from hclsm_amd.kernels import residual_rms_norm
    g = np.random.default_rng(7)
    x, r, w, gy, gh = (np.float64(np.float32(t)) for t in (g.normal(size=(6, 50)), g.normal(size=(6, 50)), g.normal(size=50),
                                                          g.normal(size=(6, 50)), g.normal(size=(6, 50))))
    t = [torch.tensor(a, dtype=F32).cuda().requires_grad_() for a in (x, r, w)]
    grads = torch.autograd.grad(residual_rms_norm(*t, eps=1e-3), t, [torch.tensor(a, dtype=F32).cuda() for a in (gy, gh)])
    f = lambda x, r, w: (gy * on.rms_norm(x + r, w, 1e-3)).sum() + (gh * (x + r)).sum()
    ins = [x, r, w]
    for i in range(3):
        d = g.normal(size=ins[i].shape)
        hi, lo = (f(*[a + s * 1e-5 * d if j == i else a for j, a in enumerate(ins)]) for s in (1, -1))
        got = (_np(grads[i]) * d).sum()
        # float32 gradients (1e-6 of their size) and differences of the third order (1e-10)
        assert abs(got - (hi - lo) / 2e-5) <= 1e-5 * np.linalg.norm(_np(grads[i])) * np.linalg.norm(d)


def test_captured_and_replayed_and_two_streams():
    from hclsm_amd.kernels import residual_rms_norm, residual_rms_norm_fp8
    x, r, w, gy, gh = _inputs((300, 768), BF16, BF16, F32, 8)
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]

    def work(ls):
        o = residual_rms_norm(*ls)
        g = torch.autograd.grad(o, ls, (gy, gh))
        with torch.no_grad():
            y8, s, _ = residual_rms_norm_fp8(*ls, group=128)
        return [t.detach() for t in o] + list(g) + [y8.float(), s]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(leaves)
        work(leaves)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = work(leaves)
    for seed in range(3):
        with torch.no_grad():
            for t in leaves:
                t.copy_(torch.randn(t.shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in res]
        for a, b in zip(got, work([t.detach().clone().requires_grad_() for t in leaves])):
            assert torch.equal(a, b)
    ref = work([t.detach().clone().requires_grad_() for t in leaves])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(work([t.detach().clone().requires_grad_() for t in leaves]))
    torch.cuda.synchronize()
    for o in outs:
        for a, b in zip(o, ref):
            assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """Rows 2^27 elements apart, and more than 2^31 elements written."""
    from hclsm_amd.kernels import residual_rms_norm
    base = torch.zeros(20, 1 << 27, dtype=BF16, device="cuda")
    x = base[:, :64]
    x.copy_(torch.randn(20, 64, device="cuda"))
    assert torch.equal(residual_rms_norm(x)[0], residual_rms_norm(x.contiguous())[0])
    del base, x
    row = torch.randn(1, 16384, device="cuda").bfloat16()
    y, h = residual_rms_norm(row.expand((1 << 17) + 3, 16384), row.expand((1 << 17) + 3, 16384))
    assert torch.equal(y, y[:1].expand_as(y)) and torch.equal(h, h[:1].expand_as(h))


def test_eight_bits_refuse_gradients():
    from hclsm_amd.kernels import residual_rms_norm_fp8
    x = torch.randn(2, 64, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        residual_rms_norm_fp8(x)
    with pytest.raises(ValueError, match="group"):
        residual_rms_norm_fp8(x.detach(), group=48)
    with pytest.raises(ValueError, match="group"):
        residual_rms_norm_fp8(torch.randn(2, 72, device="cuda"), group=32)
