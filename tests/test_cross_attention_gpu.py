"""GPU parity of cross_attention against oracle/heads.py (float64), elementwise within the bounds derived in
cross_attention_bounds.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cross_attention_bounds import assert_within, bounds
from oracle import heads as oh

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _np(t):
    return t.detach().double().cpu().numpy()


def _data(B, Lq, Lk, H, Hk, dh, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g).to(dtype)
    return rnd(B, Lq, H, dh), rnd(B, Lk, Hk, dh), rnd(B, Lk, Hk, dh), rnd(B, Lq, H, dh)


def _compare(q, k, v, g, live, dtype, what, scale=None, alive_q=None, **masks):
    """Forward and backward on the GPU against the oracle; live (B, Lk), alive_q (B, Lq) booleans."""
    from hclsm_amd.kernels import cross_attention
    ins = [t.cuda().requires_grad_() for t in (q, k, v)]
    out, lse = cross_attention(*ins, scale=scale, return_lse=True, **masks)
    grads = torch.autograd.grad(out, ins, g.cuda())
    with torch.no_grad():
        assert torch.equal(cross_attention(*ins, scale=scale, **masks), out), f"{what}: without gradients"
    qn, kn, vn, gn = (_np(t) for t in (q, k, v, g))
    dead = np.zeros(q.shape[:2], bool) if alive_q is None else ~alive_q
    qn, gn = np.where(dead[..., None, None], 0, qn), np.where(dead[..., None, None], 0, gn)
    ro, rl = oh.cross_attention(qn, kn, vn, live, scale)
    ro = np.where(dead[..., None, None], 0, ro)
    rg = oh.cross_attention_grads(qn, kn, vn, live, gn, scale)
    kz, vz = (np.where(live[:, :, None, None], t, 0) for t in (kn, vn))
    bs = bounds(qn, kz, vz, live, gn, scale, dtype)
    for name, got, ref, b in zip(("out", "dq", "dk", "dv"), (out, *grads), (ro, *rg), bs):
        assert_within(got, ref, b, f"{what} {name}")
    rl = np.where(dead[:, None, :], -np.inf, rl)
    fin = np.isfinite(rl)
    got = _np(lse)
    assert np.array_equal(np.isfinite(got), fin) and np.isneginf(got[~fin]).all(), f"{what} lse"
    if fin.any():
        sabs = np.einsum("blhd,bmhd->bhlm", np.abs(qn), np.abs(np.repeat(kz, q.shape[2] // k.shape[2], 2)))
        sabs = sabs.max(-1) * (q.shape[-1] ** -0.5 if scale is None else scale)
        tol = 2.0 ** -24 * ((q.shape[-1] + 8) * sabs + 8 * np.abs(np.where(fin, rl, 0)) + k.shape[1] / 4 + 40)
        assert (np.abs(got[fin] - rl[fin]) <= tol[fin]).all(), f"{what} lse"
    for got, rows in ((out, dead), (grads[0], dead), (grads[1], ~live), (grads[2], ~live)):
        assert not _np(got)[rows].any(), f"{what}: rows that are not live"


SHAPES = [  # B, Lq, Lk, H, Hk, dh
    (1, 1, 1, 1, 1, 8), (2, 1, 65, 4, 4, 64), (3, 1, 200, 12, 3, 64), (1, 7, 64, 2, 1, 128), (2, 32, 196, 6, 6, 64),
    (1, 130, 63, 2, 2, 32), (2, 33, 129, 6, 2, 80), (1, 65, 257, 3, 1, 96), (1, 17, 100, 2, 2, 256),
    (1, 20, 70, 4, 2, 192), (2, 300, 5, 2, 1, 64), (1, 64, 128, 2, 2, 16), (1, 129, 33, 5, 5, 136), (1, 5, 400, 8, 1, 40),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_all_keys(shape, dtype):
    print(f"cross attention {shape} {dtype}", flush=True)
    q, k, v, g = _data(*shape, dtype, 1)
    _compare(q, k, v, g, np.ones((shape[0], shape[2]), bool), dtype, f"{shape} {dtype}")


FINE = [  # at most 16 rows to a unit, or 32 in the backward and few keys
    (2, 1, 65, 4, 4, 64), (3, 1, 200, 12, 3, 64), (1, 2, 1500, 8, 2, 128), (2, 16, 196, 3, 3, 64), (2, 32, 32, 6, 6, 64),
    (2, 13, 12, 20, 5, 80), (2, 300, 5, 2, 1, 64), (1, 129, 32, 5, 5, 136), (1, 70, 31, 2, 2, 256), (2, 40, 2, 4, 2, 96),
    (1, 100, 1, 2, 2, 32), (1, 1100, 17, 2, 2, 128),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", FINE)
def test_weights_of_few_rows_and_few_keys_keep_their_rest(shape, dtype):
    from hclsm_amd.kernels import cross_attention
    print(f"cross attention {shape} {dtype}", flush=True)
    q, k, v, g = _data(*shape, dtype, 11)
    ins = [t.cuda().requires_grad_() for t in (q, k, v)]
    out = cross_attention(*ins)
    grads = torch.autograd.grad(out, ins, g.cuda())
    vals, live = [_np(t) for t in (q, k, v)], np.ones((shape[0], shape[2]), bool)
    refs = (oh.cross_attention(*vals, live, None)[0], *oh.cross_attention_grads(*vals, live, _np(g), None))
    for name, got, ref, b in zip(("out", "dq", "dk", "dv"), (out, *grads), refs,
                                 bounds(*vals, live, _np(g), None, dtype, fine=True)):
        assert_within(got, ref, b, f"{shape} {dtype} {name}")


def test_scores_gradients_past_float16():
    """dP = +-960000, ds = 0.5 dP past 65504: inf 1 + (-inf)(-1) = inf in dq, no NaN from the rounding's rest."""
    from hclsm_amd.kernels import cross_attention
    one = torch.ones(1, 1, 1, 8)
    ins = [t.half().cuda().requires_grad_()
           for t in (0 * one, torch.cat((one, -one), 1), torch.cat((60000 * one, -60000 * one), 1))]
    dq, _, dv = torch.autograd.grad(cross_attention(*ins, scale=1.0), ins, (2 * one).half().cuda())
    assert torch.isposinf(dq).all() and torch.equal(dv, torch.full_like(dv, 1.0))


SPLIT = [  # keys of a unit shared by several workgroups, rows too in the backward; many heads to a key head
    (1, 3, 1500, 4, 2, 64), (1, 1, 5000, 8, 1, 128), (2, 16, 900, 4, 2, 32), (1, 200, 700, 2, 1, 64), (2, 150, 1000, 6, 2, 128),
    (1, 70, 600, 2, 1, 256), (1, 9, 100, 40, 1, 32), (1, 4, 90, 40, 1, 256), (1, 3, 50, 70, 1, 64), (1, 40, 300, 7, 1, 200),
    (1, 33, 530, 3, 1, 96),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SPLIT)
def test_split_keys_and_rows(shape, dtype):
    print(f"split {shape} {dtype}", flush=True)
    q, k, v, g = _data(*shape, dtype, 12)
    _compare(q, k, v, g, np.ones((shape[0], shape[2]), bool), dtype, f"{shape} {dtype}")
    lens = torch.tensor([shape[2] - 37, 3][:shape[0]])
    live = np.arange(shape[2]) < lens.numpy()[:, None]
    k[~torch.tensor(live)] = float("nan")
    _compare(q, k, v, g, live, dtype, f"{shape} {dtype} lengths", key_lens=lens.cuda())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(5, 3, 70, 4, 2, 64), (4, 40, 200, 2, 2, 32), (5, 70, 140, 3, 1, 128),
                                   (4, 1, 300, 6, 2, 64), (4, 9, 90, 2, 1, 200)])
def test_masks_lengths_and_what_masked_places_hold(shape, dtype):
    """Padding masks with an empty row, lengths 0, 1 and past the end, NaN and infinities in masked keys, dead queries
    and their gradients."""
    B, Lq, Lk, H, Hk, dh = shape
    q, k, v, g = _data(*shape, dtype, 2)
    rng = np.random.default_rng(3)
    pad = rng.random((B, Lk)) < 0.3
    pad[1] = True
    pad[2, :-1], pad[2, -1] = True, False                  # the last key alone
    lens = np.array([Lk, 0, 1, Lk // 2, Lk + 7][:B])
    qlens = np.array([Lq, 1, 0, Lq + 3, (Lq + 1) // 2][:B])
    for name in ("pad", "lens", "both"):
        print(f"masks {shape} {dtype} {name}", flush=True)
        live = np.ones((B, Lk), bool)
        masks = {}
        if name != "lens":
            live &= ~pad
            masks["key_padding_mask"] = torch.tensor(pad).cuda()
        if name != "pad":
            live &= np.arange(Lk) < lens[:, None]
            masks["key_lens"] = torch.tensor(lens, dtype=torch.int32 if name == "lens" else torch.int64).cuda()
        kk, vv, qq, gg = k.clone(), v.clone(), q.clone(), g.clone()
        kk[~torch.tensor(live)], vv[~torch.tensor(live)] = float("nan"), float("inf")
        alive = None
        if name != "lens":
            alive = np.arange(Lq) < qlens[:, None]
            masks["query_lens"] = torch.tensor(qlens).cuda()
            qq[~torch.tensor(alive)], gg[~torch.tensor(alive)] = float("inf"), float("nan")
        _compare(qq, kk, vv, gg, live, dtype, f"{shape} {dtype} {name}", alive_q=alive, **masks)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scales_and_large_scores(dtype):
    """Scores of some hundreds: the running maximum moves, weights vanish, nothing overflows."""
    q, k, v, g = _data(2, 20, 300, 2, 2, 64, dtype, 4)
    live = np.ones((2, 300), bool)
    _compare(q, k, v, g, live, dtype, "scale 1", scale=1.0)
    order = torch.argsort((q.float()[:, :1, :1] * k.float()[:, :, :1]).sum(-1), 1)          # ascending for one query
    k = torch.gather(k, 1, order.expand(-1, -1, 1)[..., None].expand(k.shape))
    _compare((q.float() * 8).to(dtype), k, v, g, live, dtype, "ascending", scale=0.5)
    _compare(q, k, v, g, live, dtype, "scale small", scale=1e-3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_broadcast_and_alignment(dtype):
    from hclsm_amd.kernels import cross_attention
    B, Lq, Lk, H, dh = 3, 21, 75, 4, 64
    q, k, v, g = _data(B, Lq, Lk, H, H, dh, dtype, 5)
    live = np.ones((B, Lk), bool)
    q, k, v, g = (t.cuda() for t in (q, k, v, g))
    base = cross_attention(q, k, v)
    kv = torch.stack((k, v), 2)
    assert torch.equal(cross_attention(q, kv[:, :, 0], kv[:, :, 1]), base)
    first = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (q, k, v)]
    assert torch.equal(cross_attention(*first), base)
    odd = [torch.cat((t[..., :1], t), -1)[..., 1:] for t in (q, k, v)]                       # rows off 16 bytes
    assert torch.equal(cross_attention(*odd), base)
    every = [torch.stack((t, t), -1).flatten(-2)[..., ::2] for t in (q, k, v)]
    assert torch.equal(cross_attention(*every), base)
    mask = torch.rand(B, 2 * Lk, generator=torch.Generator().manual_seed(6)).cuda() < 0.3
    sl = mask[:, ::2]
    assert torch.equal(cross_attention(q, k, v, key_padding_mask=sl),
                       cross_attention(q, k, v, key_padding_mask=sl.contiguous().to(torch.uint8)))
    assert torch.equal(cross_attention(q, k, v, key_padding_mask=sl.float()),
                       cross_attention(q, k, v, key_padding_mask=sl))
    # learned queries repeated over the batch, one encoder state for all of them: gradients add up over the batch
    q1 = q[:1].clone().requires_grad_()
    k1, v1 = k[:1].clone().requires_grad_(), v[:1].clone().requires_grad_()
    out = cross_attention(q1.expand(B, -1, -1, -1), k1.expand(B, -1, -1, -1), v1.expand(B, -1, -1, -1))
    dq, dk, dv = torch.autograd.grad(out, (q1, k1, v1), g)
    rep = [_np(t).repeat(B, 0) for t in (q1, k1, v1)]
    ref = oh.cross_attention_grads(*rep, live, _np(g))
    bs = bounds(*rep, live, _np(g), None, dtype)
    eps = torch.finfo(dtype).eps
    for name, got, r, b in zip(("dq", "dk", "dv"), (dq, dk, dv), ref, bs[1:]):
        total = np.abs(r).sum(0, keepdims=True)                # torch's sum over the batch rounds to the type
        assert_within(got, r.sum(0, keepdims=True), b.sum(0, keepdims=True) + eps * total, f"repeated {name}")
    # a gradient of stride 0
    ql = q.clone().requires_grad_()
    (gq,) = torch.autograd.grad(cross_attention(ql, k, v).sum(), ql)
    assert torch.equal(gq, torch.autograd.grad(cross_attention(ql, k, v), ql, torch.ones_like(base))[0])


def test_gradients_against_differences():
    """<gradient, direction> of the float32 kernels against central differences of the float64 statement."""
    q, k, v, g = _data(2, 9, 70, 4, 2, 32, torch.float32, 7)
    from hclsm_amd.kernels import cross_attention
    lens = torch.tensor([70, 33])
    live = np.arange(70) < lens.numpy()[:, None]
    ins = [t.cuda().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(cross_attention(*ins, key_lens=lens.cuda()), ins, g.cuda())
    vals = [_np(t) for t in (q, k, v)]
    bs = bounds(*vals, live, _np(g))
    f = lambda *t: (_np(g) * oh.cross_attention(*t, live)[0]).sum()
    rng, h = np.random.default_rng(8), 1e-5
    for i in range(3):
        u = rng.normal(size=vals[i].shape)
        up, dn = list(vals), list(vals)
        up[i], dn[i] = vals[i] + h * u, vals[i] - h * u
        diff = (f(*up) - f(*dn)) / (2 * h)
        assert abs((_np(grads[i]) * u).sum() - diff) <= (bs[1 + i] * np.abs(u)).sum() + 1e-7 * abs(diff)


def test_empty_sizes():
    from hclsm_amd.kernels import cross_attention
    for B, Lq, Lk, H in ((0, 3, 4, 2), (2, 0, 4, 2), (2, 3, 0, 2)):
        q = torch.randn(B, Lq, H, 16, device="cuda", requires_grad=True)
        k, v = (torch.randn(B, Lk, 1, 16, device="cuda", requires_grad=True) for _ in range(2))
        out, lse = cross_attention(q, k, v, return_lse=True)
        grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
        assert out.shape == q.shape and lse.shape == (B, H, Lq)
        assert [t.shape for t in grads] == [q.shape, k.shape, v.shape]
        if Lk == 0:
            assert not out.any() and torch.isneginf(lse).all() and not grads[0].any()
        if Lq == 0:
            assert not grads[1].any() and not grads[2].any()
    for dh in (16, 256):                  # no query head; queries of length zero
        for Lq, H in ((3, 0), (0, 2)):
            q = torch.empty(2, Lq, H, dh, device="cuda", requires_grad=True)
            k, v = (torch.randn(2, 70, 2, dh, device="cuda", requires_grad=True) for _ in range(2))
            out = cross_attention(q, k, v)
            grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
            assert out.shape == q.shape and not grads[1].any() and not grads[2].any()


def test_same_bits_partial_gradients_and_side_stream():
    from hclsm_amd.kernels import cross_attention
    q, k, v, g = (t.cuda() for t in _data(2, 50, 300, 4, 2, 64, torch.bfloat16, 9))
    ins = [t.clone().requires_grad_() for t in (q, k, v)]
    out = cross_attention(*ins)
    first = torch.autograd.grad(out, ins, g, retain_graph=True)
    again = torch.autograd.grad(out, ins, g)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    for Lq in (50, 5):                    # tiles of rows, and few rows
        qs, gs = q[:, :Lq].contiguous(), g[:, :Lq].contiguous()
        ref = torch.autograd.grad(cross_attention(qs.requires_grad_(), *ins[1:]), [qs, *ins[1:]], gs)
        for i in range(3):                # a frozen encoder, learned keys: gradients of one input alone
            parts = [qs.detach(), k, v]
            parts[i] = parts[i].clone().requires_grad_()
            (one,) = torch.autograd.grad(cross_attention(*parts), parts[i], gs)
            assert torch.equal(one, ref[i])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2 = cross_attention(q, k, v)
    side.synchronize()
    assert torch.equal(o2, out)


def test_graph_replays():
    """Forward and backward captured (fresh leaves, no eager graph of them alive) and replayed on new data, eager work
    between the replays."""
    from hclsm_amd.kernels import cross_attention
    for Lq in (1, 40):
        q, k, v, g = (t.cuda() for t in _data(2, Lq, 700, 4, 2, 64, torch.bfloat16, 10))
        lens = torch.tensor([700, 300], device="cuda")

        def step(leaves):
            out = cross_attention(*leaves, key_lens=lens)
            return (out.detach(), *torch.autograd.grad(out, leaves, g))

        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(leaves)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(leaves)
        for seed in range(3):
            gen = torch.Generator("cuda").manual_seed(seed)
            with torch.no_grad():
                for t in leaves:
                    t.normal_(generator=gen)
            g.normal_(generator=gen)
            lens.copy_(torch.tensor([650 - 100 * seed, seed], device="cuda"))
            graph.replay()
            torch.cuda.synchronize()
            ref = step([t.detach().clone().requires_grad_() for t in leaves])
            assert all(torch.equal(a, b) for a, b in zip(got, ref)), f"replay {seed} of Lq {Lq}"
        del graph


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_rotation_and_attention_together(dtype):
    """As a block uses them: norm and rotation of queries and keys, attention, and the gradients back through all of it.
    Each stage is checked on what it was given."""
    from hclsm_amd.kernels import RotaryPlan, cross_attention, qk_norm_rotary
    q, k, v, g = (t.cuda() for t in _data(2, 40, 150, 6, 2, 64, dtype, 11))
    wq, wk = (1 + 0.1 * torch.randn(64, generator=torch.Generator().manual_seed(i)).cuda() for i in range(2))
    leaves = [t.requires_grad_() for t in (q, k, v, wq, wk)]
    plan = RotaryPlan(32, layout="interleaved")
    kpos = torch.arange(150, device="cuda") * 3
    lens = torch.tensor([150, 64], device="cuda")
    qr, kr = qk_norm_rotary(q, k, wq, wk, plan, None, kpos)
    out = cross_attention(qr, kr, v, key_lens=lens)
    dqr, dkr, *grads = torch.autograd.grad(out, [qr, kr] + leaves, g)
    live = np.arange(150) < lens.cpu().numpy()[:, None]
    vals = [_np(t) for t in (qr, kr, v)]
    refs = (oh.cross_attention(*vals, live)[0], *oh.cross_attention_grads(*vals, live, _np(g)))
    for name, got, ref, b in zip(("out", "dq", "dk", "dv"), (out, dqr, dkr, grads[2]), refs,
                                 bounds(*vals, live, _np(g), None, dtype)):
        assert_within(got, ref, b, name)
    freq, eps = plan.inv_freq.numpy(), torch.finfo(dtype).eps / 2
    for name, x, w, go, p, y, gx, gw in (("q", q, wq, dqr, np.arange(40), qr, grads[0], grads[3]),
                                         ("k", k, wk, dkr, kpos.cpu().numpy(), kr, grads[1], grads[4])):
        ref = oh.norm_rotate(_np(x), _np(w), p, freq, 1.0, "interleaved")
        rx, rw = oh.norm_rotate_grads(_np(x), _np(w), _np(go), p, freq, 1.0, "interleaved")
        # the norm's own roundings: 24 (forward), 72 and 400 units (test_norm_rotary_gpu.py) of terms at most 64 times
        # the largest element of a row
        big = lambda t: np.abs(t).max(-1, keepdims=True)
        r = 1 / np.sqrt((_np(x) ** 2).mean(-1, keepdims=True))
        n = big(_np(x)) * r
        assert_within(y, ref, eps * np.abs(ref) + 48 * 2.0 ** -24 * n * np.abs(_np(w)).max(), name + " normed")
        d = 2 * big(_np(go))
        assert_within(gx, rx, eps * np.abs(rx) + 72 * 2.0 ** -24 * r * d * np.abs(_np(w)).max() * (1 + n * n), "d" + name)
        assert_within(gw, rw, 400 * 2.0 ** -24 * (d * n).sum((0, 1, 2)) + 2.0 ** -23 * np.abs(rw), "dw" + name)


def test_second_derivatives_are_refused():
    from hclsm_amd.kernels import RotaryPlan, cross_attention, qk_norm_rotary, rotary_embedding
    x = torch.randn(1, 4, 2, 16, device="cuda", requires_grad=True)
    plan = RotaryPlan(16)
    for f in (lambda x: cross_attention(x, x, x), lambda x: qk_norm_rotary(x, None, None, None, plan)[0],
              lambda x: rotary_embedding(x, plan)):
        y = f(x)
        (g,) = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
        first = torch.autograd.grad(f(x), x, torch.ones_like(y))[0]
        assert torch.equal(g, first)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)


def test_offsets_past_32_bits():
    """Keys and values of 4.6 GB each: the last keys of a long cache, for one query and for a tile of them, forward and
    backward, and the rotation of as long a tensor."""
    from hclsm_amd.kernels import RotaryPlan, cross_attention, rotary_embedding
    L, Hk, dh, n = 2_200_013, 8, 128, 100
    gen = torch.Generator("cuda").manual_seed(13)
    k = torch.zeros(1, L, Hk, dh, dtype=torch.bfloat16, device="cuda")
    v = torch.full_like(k, float("nan"))
    tail = [torch.randn(1, n, Hk, dh, generator=gen, device="cuda").bfloat16() for _ in range(2)]
    k[:, -n:], v[:, -n:] = tail
    pad = torch.ones(1, L, dtype=torch.bool, device="cuda")
    pad[:, -n:] = False
    for Lq in (1, 40):
        print(f"offsets past 32 bits, {Lq} queries", flush=True)
        q = torch.randn(1, Lq, Hk, dh, generator=gen, device="cuda").bfloat16()
        g = torch.randn(q.shape, generator=gen, device="cuda").bfloat16()
        live = np.ones((1, n), bool)
        vals = [_np(t) for t in (q, *tail)]
        refs = (oh.cross_attention(*vals, live)[0], *oh.cross_attention_grads(*vals, live, _np(g)))
        ins = [t.requires_grad_() for t in (q, k, v)]
        out = cross_attention(*ins, key_padding_mask=pad)
        dq, dk, dv = torch.autograd.grad(out, ins, g)
        assert not dk[:, :-n].any() and not dv[:, :-n].any()
        for name, got, ref, b in zip(("out", "dq", "dk", "dv"), (out, dq, dk[:, -n:], dv[:, -n:]), refs,
                                     bounds(*vals, live, _np(g), None, torch.bfloat16)):
            assert_within(got, ref, b, f"{Lq} queries {name}")
        del out, dq, dk, dv
    plan = RotaryPlan(dh)
    with torch.no_grad():
        k[:, -n:] = tail[0]
        y = rotary_embedding(k, plan)[:, -n:]
        assert torch.equal(y, rotary_embedding(tail[0], plan, torch.arange(L - n, L, device="cuda")))


def test_two_streams_at_once():
    """Calls on two streams in flight together, each with a workspace of its own (keys split, partial gradients)."""
    from hclsm_amd.kernels import cross_attention
    data = [_data(1, Lq, 3000, 4, 2, 64, torch.bfloat16, 20 + Lq) for Lq in (2, 90)]
    sets = [[t.cuda() for t in d] for d in data]

    def step(q, k, v, g):
        ins = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        out = cross_attention(*ins)
        return (out.detach(), *torch.autograd.grad(out, ins, g))

    refs = [step(*d) for d in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got[i].append(step(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, refs[i]))
