"""GPU parity of linear attention with decays against oracle/linear_attention.py (float64), elementwise.

Tolerances: half a step of the output type at the value (finfo.eps / 2), plus a share of M, the same sum over the magnitudes of
all its terms (the oracle on absolute values).  A value in N bf16 parts is off by at most 2^-8N of itself, products leave out
what lies below the last part.
  Outputs of 16-bit inputs: the pair's product (float16: its two low parts) 2^-16, the weight in two parts 2^-16, its product
  2^-16, or the state in two parts 2^-16 and its product 2^-16: 3 * 2^-16.  Of float32 inputs, in three parts: three products
  left out at 2^-24 each for both factors, and the parts themselves, for each of two products in a row: 16 * 2^-24.
  States: X in three parts and the products left out: 8 * 2^-24.
  Float32 sums and powers: at most dk + dv + 64 additions inside a chunk, one for each token in the state, two roundings a chunk
  and segment for the decay, 8 for the powers: (dk + dv + L + 128) * 2^-24.
Sums over shared heads add at most 16 roundings of 2^-24, inside the same allowance.
float32 has no value below 2^-149 and powers below 2^-126 may be zero, with which at most 16 terms of at most 4 are lost here: results
are off by up to 2^-120 besides (float16: by half its smallest step)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import linear_attention as ol

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -120, torch.bfloat16: 2.0 ** -120, torch.float16: 2.0 ** -25}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _within(got, ref, M, share, what):
    got_, dt = _np(got), got.dtype
    tol = torch.finfo(dt).eps / 2 * np.abs(ref) + share * M * (1 + torch.finfo(dt).eps) + TINY[dt]
    assert got_.shape == ref.shape, f"{what}: {got_.shape} for {ref.shape}"
    assert np.isfinite(got_).all(), f"{what}: not finite"
    err = np.abs(got_ - ref)
    assert (err <= tol).all(), f"{what}: {(err - tol).max():.3e} over at {np.unravel_index((err - tol).argmax(), err.shape)}"


def _shares(dtype, L, dk, dv):
    sums = (dk + dv + L + 128) * U
    return (16 * U if dtype == F32 else 3 * 2.0 ** -16) + sums, 8 * U + sums


def _inputs(B, L, H, Hk, dk, dv, dtype, seed=0, state=True):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(*s, generator=g).to(dtype) for s in ((B, L, H, dk), (B, L, Hk, dk), (B, L, Hk, dv)))
    s0 = 2.0 * torch.randn(B, H, dk, dv, generator=g) if state else None
    go, gs = torch.randn(B, L, H, dv, generator=g).to(dtype), torch.randn(B, H, dk, dv, generator=g) if state else None
    decay = -torch.tensor([0.02, 0.0, 0.7, 0.002, 3.0])[torch.arange(H) % 5]
    return q, k, v, s0, decay, go, gs


def _compare(q, k, v, s0, decay, go, gs, lens=None, scale=None, outs=None, lens_gpu=None):
    """Forward and all gradients through both outputs against the oracle."""
    from hclsm_amd.kernels import linear_attention
    B, L, H, dk = q.shape
    dv = v.shape[3]
    c = dk ** -0.5 if scale is None else scale
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)] + ([s0.cuda().requires_grad_()] if s0 is not None else [])
    n = lens_gpu if lens_gpu is not None else None if lens is None else torch.tensor(lens, dtype=torch.int32).cuda()
    out, s1 = linear_attention(*leaves[:3], decay.cuda(), initial_state=leaves[3] if s0 is not None else None, seq_lens=n,
                               scale=scale, return_state=True)
    up = [go.cuda()] + ([gs.cuda()] if gs is not None else [])
    grads = torch.autograd.grad((out, s1) if gs is not None else (out,), leaves, up)
    a = [_np(t) for t in (q, k, v)]
    m = [np.abs(t) for t in a]
    share, state = _shares(q.dtype, L, dk, dv)
    ref, M = ol.linear_attention(*a, _np(decay), c, _np(s0), lens), \
        ol.linear_attention(*m, _np(decay), c, None if s0 is None else np.abs(_np(s0)), lens)
    _within(out, ref[0], M[0], share, "out")
    _within(s1, ref[1], M[1], state, "state")
    rg = ol.linear_attention_grads(*a, _np(decay), c, _np(go), _np(s0), _np(gs), lens)
    mg = ol.linear_attention_grads(*m, _np(decay), c, np.abs(_np(go)), None if s0 is None else np.abs(_np(s0)),
                                   None if gs is None else np.abs(_np(gs)), lens)
    for name, got, r, M in zip(("dq", "dk", "dv", "dstate"), grads, rg, mg):
        _within(got, r, M, state if name == "dstate" else share, name)
    return out, s1, grads


SHAPES = [  # B, L, H, Hk, dk, dv
    (1, 1, 1, 1, 8, 8), (2, 2, 3, 3, 16, 24), (1, 31, 2, 1, 32, 64), (2, 63, 2, 2, 64, 64), (1, 64, 5, 5, 64, 72),
    (1, 65, 2, 2, 96, 128), (2, 130, 4, 2, 48, 96), (1, 70, 2, 1, 256, 256), (1, 97, 1, 1, 136, 40), (3, 5, 6, 6, 64, 64),
    (1, 200, 16, 4, 24, 200), (1, 33, 2, 2, 64, 192), (1, 300, 1, 1, 128, 128),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(shape, dtype):
    print(f"linear attention {shape} {dtype}", flush=True)
    _compare(*_inputs(*shape, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("state", [False, True])
def test_split_over_time(dtype, state):
    """Few heads and many tokens: segments, with lengths that end in the first, in the middle, on a border and at the end."""
    from hclsm_amd import _lib
    B, L, H, dk, dv = 4, 1500, 2, 64, 32
    code = {F32: 0, BF16: 1, F16: 2}[dtype]
    for bwd in (0, 1):
        assert _lib.lib().hclsm_linear_attention_workspace(B, L, H, H, dk, dv, code, bwd) > 0
    ins = list(_inputs(B, L, H, H, dk, dv, dtype, 3, state))
    print(f"split {dtype} {state}", flush=True)
    _compare(*ins)
    _compare(*ins, lens=[7, 1500, 0, 768])
    ins[4] = torch.tensor([0.0, -1e-4])
    _compare(*ins, lens=[1499, 256, 1, 1025])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("i64", [False, True])
def test_lengths_and_what_lies_behind_them(dtype, i64):
    """Rows of no token, lengths below zero and past the end; NaN and infinities behind the live tokens reach nothing."""
    B, L, H, Hk, dk, dv = 6, 150, 4, 2, 32, 40
    q, k, v, s0, decay, go, gs = _inputs(B, L, H, Hk, dk, dv, dtype, 5)
    lens = [0, 150, 64, 77, -3, 1 << 20]
    n = torch.tensor([0, 150, 64, 77, -3, 1 << 20], dtype=torch.int64 if i64 else torch.int32)
    clean = _compare(q, k, v, s0, decay, go, gs, lens=lens, lens_gpu=n.cuda())
    wide = torch.stack((n, n + 1), 1).cuda()[:, 0]
    for t in (q, k, v, go):
        for b, m in enumerate(lens):
            t[b, max(m, 0):] = float("nan")
            t[b, max(m, 0)::2] = float("inf")
    from hclsm_amd.kernels import linear_attention
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, s0)]
    out = linear_attention(*leaves[:3], decay.cuda(), initial_state=leaves[3], seq_lens=wide, return_state=True)
    grads = torch.autograd.grad(out, leaves, (go.cuda(), gs.cuda()))
    for a, b in zip(out + grads, (clean[0], clean[1]) + clean[2]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_extreme_decays(dtype):
    """No memory (-inf, and far below float32's exponents), no decay, and memories of a few tokens."""
    ins = list(_inputs(2, 140, 6, 6, 32, 32, dtype, 6))
    ins[4] = torch.tensor([float("-inf"), -1e30, -200.0, 0.0, -12.0, -1e-7])
    _compare(*ins)
    from hclsm_amd.kernels import linear_attention
    q, k, v = (t.cuda() for t in ins[:3])
    got = linear_attention(q, k, v, ins[4].cuda(), scale=1.0)
    alone = (q.double() * k.double()).sum(-1, keepdim=True) * v.double()
    M = (q.double() * k.double()).abs().sum(-1, keepdim=True) * v.double().abs()
    _within(got[:, :, :2], _np(alone[:, :, :2]), _np(M[:, :, :2]), _shares(dtype, 0, 32, 32)[0], "no memory")


def test_scales_and_sizes_of_values():
    """float16 values whose pairs pass 65504, and scales far from one: no intermediate has float16's range."""
    q, k, v, s0, decay, go, gs = _inputs(1, 100, 2, 2, 64, 64, F16, 7)
    q, k, v, go = 64 * q, 64 * k, v / 512, go / 64
    _compare(q, k, v, 1000 * s0, decay, go, gs, scale=2.0 ** -10)
    _compare(q.bfloat16(), k.bfloat16(), v.bfloat16() * 1e20, s0, decay, go.bfloat16(), gs, scale=1e-12)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_alignment_and_broadcast(dtype):
    """Views of one projection, heads first, rows at odd addresses, a batch and heads repeated by stride 0."""
    from hclsm_amd.kernels import linear_attention
    g = torch.Generator().manual_seed(8)
    B, L, H, d = 2, 70, 3, 64
    decay = torch.tensor([-0.1, -0.01, 0.0]).cuda()
    fused = torch.randn(B, L, 3, H, d, generator=g).to(dtype).cuda()
    first = torch.randn(3, B, H, L, d, generator=g).to(dtype).cuda()
    odd = torch.randn(3, B, L, H, d + 1, generator=g).to(dtype).cuda()
    one = torch.randn(3, 1, L, 1, d, generator=g).to(dtype).cuda()
    far = torch.randn(3, B, L, H, 2 * d, generator=g).to(dtype).cuda()
    views = {"fused": [fused[:, :, i] for i in range(3)], "heads first": [first[i].transpose(1, 2) for i in range(3)],
             "odd": [odd[i, ..., 1:] for i in range(3)], "repeated": [one[i].expand(B, L, H, d) for i in range(3)],
             "strided": [far[i, ..., ::2] for i in range(3)]}
    share, _ = _shares(dtype, L, d, d)
    for name, (q, k, v) in views.items():
        print(f"strides {name} {dtype}", flush=True)
        a = [_np(t) for t in (q, k, v)]
        M, _ = ol.linear_attention(*(np.abs(t) for t in a), _np(decay), d ** -0.5)
        _within(linear_attention(q, k, v, decay), ol.linear_attention(*a, _np(decay), d ** -0.5)[0], M, share, name)
    # the gradient of a view, an output gradient of stride 0, and decays that are a view
    x = fused.clone().requires_grad_()
    y = linear_attention(x[:, :, 0], x[:, :, 1], x[:, :, 2], torch.stack((decay, decay), 1)[:, 0])
    (gx,) = torch.autograd.grad(y.sum(), x)
    a = [_np(fused[:, :, i]) for i in range(3)]
    ones = np.ones((B, L, H, d))
    ref = ol.linear_attention_grads(*a, _np(decay), d ** -0.5, ones)
    mag = ol.linear_attention_grads(*(np.abs(t) for t in a), _np(decay), d ** -0.5, ones)
    for i in range(3):
        _within(gx[:, :, i], ref[i], mag[i], share, f"gradient of view {i}")


def test_some_gradients_alone():
    """Only what requires a gradient is formed, and is the same as with all; one output's gradient alone; none at all."""
    from hclsm_amd.kernels import linear_attention
    q, k, v, s0, decay, go, gs = (t.cuda() for t in _inputs(2, 80, 4, 2, 32, 64, BF16, 9))

    def grads(need, use=(True, True)):
        t = [x.clone().requires_grad_(bool(n)) for x, n in zip((q, k, v, s0), need)]
        o = linear_attention(*t[:3], decay, initial_state=t[3], return_state=True)
        outs = [x for x, u in zip(o, use) if u]
        got = iter(torch.autograd.grad(outs, [x for x in t if x.requires_grad], [x for x, u in zip((go, gs), use) if u],
                                       allow_unused=True))
        return [next(got) if n else None for n in need]
    full = grads((1, 1, 1, 1))
    for i in range(4):
        need = [j == i for j in range(4)]
        assert torch.equal(grads(need)[i], full[i]), i
    state = grads((1, 1, 1, 1), (False, True))
    assert not state[0].any()
    r = ol.linear_attention_grads(*(_np(t) for t in (q, k, v)), _np(decay), 32 ** -0.5, np.zeros(go.shape), _np(s0), _np(gs))
    m = ol.linear_attention_grads(*(np.abs(_np(t)) for t in (q, k, v)), _np(decay), 32 ** -0.5, np.zeros(go.shape),
                                  np.abs(_np(s0)), np.abs(_np(gs)))
    for name, got, ref, M in zip(("dk", "dv", "dstate"), state[1:], r[1:], m[1:]):
        _within(got, ref, M, _shares(BF16, 80, 32, 64)[0], name)
    with pytest.raises(RuntimeError):       # no second derivative
        t = q.clone().requires_grad_()
        (g1,) = torch.autograd.grad(linear_attention(t, k, v, decay).sum(), t, create_graph=True)
        g1.sum().backward()


def test_gradients_against_differences():
    """<gradient, direction> of the float32 kernels against central differences of the float64 statement."""
    from hclsm_amd.kernels import linear_attention
    r = np.random.default_rng(10)
    q, k, v, s0 = (np.float64(np.float32(r.normal(size=s))) for s in ((2, 40, 4, 16), (2, 40, 2, 16), (2, 40, 2, 24), (2, 4, 16, 24)))
    go, gs = (np.float64(np.float32(r.normal(size=s))) for s in ((2, 40, 4, 24), (2, 4, 16, 24)))
    decay = np.float64(np.float32([-0.05, 0.0, -0.5, -2.0]))
    t = [torch.tensor(x, dtype=F32).cuda().requires_grad_() for x in (q, k, v, s0)]
    o = linear_attention(*t[:3], torch.tensor(decay, dtype=F32).cuda(), initial_state=t[3], return_state=True, scale=0.25)
    grads = torch.autograd.grad(o, t, [torch.tensor(x, dtype=F32).cuda() for x in (go, gs)])

    def f(x):
        y, s = ol.linear_attention(*x[:3], decay, 0.25, x[3])
        return (go * y).sum() + (gs * s).sum()
    x = [q, k, v, s0]
    for i in range(4):
        d = r.normal(size=x[i].shape)
        h = 1e-4
        num = (f([y + h * d if j == i else y for j, y in enumerate(x)]) - f([y - h * d if j == i else y for j, y in enumerate(x)])) / (2 * h)
        # the sum is of degree two or less in any one input: differences are exact but for float64's rounding
        got = (_np(grads[i]) * d).sum()
        assert abs(got - num) <= 1e-5 * np.linalg.norm(_np(grads[i])) * np.linalg.norm(d), (i, got, num)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 8, 8), (3, 4, 2, 64, 64), (2, 6, 6, 96, 80), (2, 2, 1, 256, 256), (5, 3, 3, 136, 24), (1, 2, 2, 16, 200)])
def test_step(shape, dtype):
    """One token, the state in place; strided tokens of a fused projection."""
    from hclsm_amd.kernels import linear_attention_step
    B, H, Hk, dk, dv = shape
    print(f"step {shape} {dtype}", flush=True)
    q, k, v, s0, decay, _, _ = _inputs(B, 1, H, Hk, dk, dv, dtype, 11)
    a = [_np(t) for t in (q, k, v)]
    ref = ol.linear_attention(*a, _np(decay), dk ** -0.5, _np(s0))
    M = ol.linear_attention(*(np.abs(t) for t in a), _np(decay), dk ** -0.5, np.abs(_np(s0)))
    state = s0.cuda()
    wide = torch.zeros(B, H * dk + Hk * (dk + dv) + 1, dtype=dtype, device="cuda")[:, 1:]     # rows at odd addresses
    tq, tk, tv = (t.unflatten(1, s) for t, s in zip(wide.split((H * dk, Hk * dk, Hk * dv), 1), ((H, dk), (Hk, dk), (Hk, dv))))
    for t, x in ((tq, q), (tk, k), (tv, v)):
        t.copy_(x[:, 0])
    out = linear_attention_step(tq, tk, tv, decay.cuda(), state)
    # three roundings of a state's element (power, product, sum), dk products and sums of the output
    _within(state, ref[1], M[1], 6 * U, "state")
    _within(out, ref[0][:, 0], M[0][:, 0], (dk + 10) * U, "out")


@pytest.mark.parametrize("i64", [False, True])
def test_step_rows_of_a_pool(i64):
    """States by index, padding rows, and every other state left as it was."""
    from hclsm_amd.kernels import linear_attention_step
    B, N, H, dk, dv = 7, 9, 2, 32, 64
    q, k, v, _, decay, _, _ = _inputs(B, 1, H, H, dk, dv, BF16, 12)
    q, k, v = (t[:, 0].cuda() for t in (q, k, v))
    base = torch.randn(N, H + 1, dk, dv, generator=torch.Generator().manual_seed(1)).cuda()
    rows = torch.tensor([8, -1, 0, 5, N, 2, 1 << 30], dtype=torch.int64 if i64 else torch.int32).cuda()
    pool = base.clone()
    out = linear_attention_step(q, k, v, decay.cuda(), pool[:, :H], rows=torch.stack((rows, rows), 1)[:, 1])
    live = [0, 2, 3, 5]
    at = rows[live].long()
    want = base[at, :H].contiguous()
    o = linear_attention_step(q[live], k[live], v[live], decay.cuda(), want)
    assert torch.equal(out[live], o) and not out[[1, 4, 6]].any()
    ref = base.clone()
    ref[at, :H] = want
    assert torch.equal(pool, ref)
    assert not linear_attention_step(q, k, v, decay.cuda(), base[:0, :H], rows=rows).any()      # no state at all


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_prompt_then_tokens(dtype):
    """A prompt in two parts of different lengths, then single tokens, are the whole sequence."""
    from hclsm_amd.kernels import linear_attention, linear_attention_step
    B, L, H, dk, dv = 2, 90, 3, 64, 64
    q, k, v, _, decay, _, _ = _inputs(B, L, H, H, dk, dv, dtype, 13, False)
    a = [_np(t) for t in (q, k, v)]
    ref, end = ol.linear_attention(*a, _np(decay), dk ** -0.5)
    M, Me = ol.linear_attention(*(np.abs(t) for t in a), _np(decay), dk ** -0.5)
    q, k, v, decay = (t.cuda() for t in (q, k, v, decay))
    share, state = _shares(dtype, L, dk, dv)
    first = torch.tensor([70, 33], dtype=torch.int32).cuda()
    o1, s = linear_attention(q[:, :70], k[:, :70], v[:, :70], decay, seq_lens=first, return_state=True)
    _within(o1[0], ref[0, :70], M[0, :70], share, "first part")
    _within(o1[1, :33], ref[1, :33], M[1, :33], share, "first part")
    # the second part starts where each row's first ended
    pick = lambda t: torch.stack((t[0, 70:80], t[1, 33:43]))
    o2, s = linear_attention(pick(q), pick(k), pick(v), decay, initial_state=s, return_state=True)
    for b, at in ((0, 70), (1, 33)):
        _within(o2[b], ref[b, at:at + 10], M[b, at:at + 10], share, "second part")
    for t in range(10):
        at = (80 + t, 43 + t)
        tok = lambda x: torch.stack((x[0, at[0]], x[1, at[1]]))
        o = linear_attention_step(tok(q), tok(k), tok(v), decay, s)
        for b in range(2):
            _within(o[b], ref[b, at[b]], M[b, at[b]], share, f"token {t}")
    _within(s[0], end[0], Me[0], state, "last state")


def test_nothing_to_do():
    from hclsm_amd.kernels import linear_attention, linear_attention_step
    d = torch.zeros(3, device="cuda")
    s0 = torch.randn(2, 3, 16, 24, device="cuda", requires_grad=True)
    e = torch.empty(2, 0, 3, 16, device="cuda", requires_grad=True)
    out, s1 = linear_attention(e, e, e.new_empty(2, 0, 3, 24), d, initial_state=s0, return_state=True)
    assert out.shape == (2, 0, 3, 24) and torch.equal(s1, s0)
    ge, gs = torch.autograd.grad(s1, (e, s0), 2.0 * s0.detach(), allow_unused=True)
    assert ge.shape == e.shape and torch.equal(gs, 2.0 * s0.detach())
    assert not linear_attention(e, e, e.new_empty(2, 0, 3, 24), d, return_state=True)[1].any()
    z = torch.empty(0, 5, 3, 16, device="cuda")
    out, s1 = linear_attention(z, z, z, d, return_state=True)
    assert out.shape == z.shape and s1.shape == (0, 3, 16, 16)
    assert linear_attention_step(z[:, 0], z[:, 0], z[:, 0], d, s1).shape == (0, 3, 16)


def test_same_bits_streams_and_two_at_once():
    """Calls on two streams side by side, each with its workspace, give the bits of calls alone."""
    from hclsm_amd.kernels import linear_attention
    sets = [[t.cuda() for t in _inputs(1, 2000, 4, 2, 64, 64, BF16, s)] for s in (20, 21)]

    def run(q, k, v, s0, decay, go, gs):
        t = [x.clone().requires_grad_() for x in (q, k, v, s0)]
        o = linear_attention(*t[:3], decay, initial_state=t[3], return_state=True)
        return tuple(x.detach() for x in o) + torch.autograd.grad(o, t, (go, gs))
    alone = [run(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = run(*sets[i])
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_captured_and_replayed():
    """Forward, backward (leaves of their own) and the step in one graph, replayed with eager work in between."""
    from hclsm_amd.kernels import linear_attention, linear_attention_step
    q, k, v, s0, decay, go, gs = (t.cuda() for t in _inputs(1, 1200, 4, 2, 64, 64, BF16, 22))
    leaves = [t.clone().requires_grad_() for t in (q, k, v, s0)]
    state = torch.zeros(1, 4, 64, 64, device="cuda")

    def work():
        o = linear_attention(*leaves[:3], decay, initial_state=leaves[3], return_state=True)
        g = torch.autograd.grad(o, leaves, (go, gs))
        state.copy_(o[1].detach())
        y = linear_attention_step(leaves[0][:, 0].detach(), leaves[1][:, 0].detach(), leaves[2][:, 0].detach(), decay, state)
        return tuple(t.detach() for t in o) + g + (y, state)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = work()
    for seed in range(3):
        gen = torch.Generator("cuda").manual_seed(seed)
        with torch.no_grad():
            for t in leaves:
                t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in res]
        t = [x.detach().clone().requires_grad_() for x in leaves]
        o = linear_attention(*t[:3], decay, initial_state=t[3], return_state=True)
        ref = [x.detach() for x in o] + list(torch.autograd.grad(o, t, (go, gs)))
        s = o[1].detach().clone()
        ref += [linear_attention_step(t[0][:, 0].detach(), t[1][:, 0].detach(), t[2][:, 0].detach(), decay, s), s]
        torch.cuda.synchronize()
        for x, y in zip(got, ref):
            assert torch.equal(x, y)


def test_offsets_past_32_bits():
    """Tokens 2^26 elements apart (9 GB of one tensor) and a state behind the first 2^31 elements of its pool."""
    from hclsm_amd.kernels import linear_attention, linear_attention_step
    L, d = 70, 16
    q, k, v, _, decay, _, _ = _inputs(1, L, 1, 1, d, d, BF16, 23, False)
    base = torch.zeros(L, 1 << 26, dtype=BF16, device="cuda")
    views = []
    for i, t in enumerate((q, k, v)):
        w = base[:, 16 * i:16 * i + d]
        w.copy_(t[0, :, 0])
        views.append(w[None, :, None])
    got = linear_attention(*views, decay.cuda())
    assert torch.equal(got, linear_attention(q.cuda(), k.cuda(), v.cuda(), decay.cuda()))
    del base, views
    pool = torch.zeros((1 << 31) // (256 * 256) + 8, 1, 256, 256, device="cuda")
    t = [torch.randn(1, 1, 256, device="cuda") for _ in range(3)]
    row = torch.tensor([pool.shape[0] - 1], device="cuda")
    out = linear_attention_step(*t, decay.cuda(), pool, rows=row)
    one = torch.zeros(1, 1, 256, 256, device="cuda")
    assert torch.equal(out, linear_attention_step(*t, decay.cuda(), one))
    assert torch.equal(pool[-1], one[0]) and not pool[:-1].any()


def test_step_refuses_gradients():
    from hclsm_amd.kernels import linear_attention_step
    x = torch.randn(1, 2, 16, device="cuda", requires_grad=True)
    s, d = torch.zeros(1, 2, 16, 16, device="cuda"), torch.zeros(2, device="cuda")
    with pytest.raises(RuntimeError, match="no gradient"):
        linear_attention_step(x, x, x, d, s)
    with torch.no_grad():
        linear_attention_step(x, x, x, d, s)


@pytest.mark.parametrize("dtype,H", [(F32, 16384 + 4), (BF16, 32768 - 4)])
def test_many_heads_of_one_token(dtype, H):
    """Tokens of 2^22 to 2^23 elements, forward and backward: some heads are as if alone."""
    from hclsm_amd.kernels import linear_attention
    L, d, some = 40, 256, [0, 1, H // 2, H - 1]
    gen = torch.Generator("cuda").manual_seed(24)
    q, k, v, go = (torch.randn(1, L, H, d, generator=gen, device="cuda", dtype=dtype) for _ in range(4))
    decay = -torch.rand(H, generator=gen, device="cuda")

    def run(q, k, v, decay, go):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = linear_attention(*leaves, decay)
        return [o.detach(), *torch.autograd.grad(o, leaves, go)]
    got = [t[:, :, some] for t in run(q, k, v, decay, go)]
    want = run(*(t[:, :, some].contiguous() for t in (q, k, v)), decay[some], go[:, :, some].contiguous())
    for a, b in zip(got, want):
        assert torch.equal(a, b)
