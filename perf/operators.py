"""Cross attention and its head-wise norms and rotations as measured cases.

    rotary   rotary_embedding: the position rotation of one tensor of heads, alone or with its gradient
    norm     qk_norm_rotary: RMS norm of queries and keys for each head and their rotation in one pass
    cross    cross_attention: queries of one length against keys and values of another (slots or goal queries
             against an encoder's tokens), alone or with the gradients of q, k and v

With ``own`` false, ``run`` computes the plain form: elementary torch operations in float32 (angles in float64),
rounded once at the end.  With ``own`` true it makes a user's calls of ``hclsm_amd.kernels``.  ``exact`` restates
each operator in float64 and takes gradients by differentiating that statement.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
_EPS = 1e-6


def listed() -> list:
    return [
        # serving, one new token for each of 64 clips, positions far into a long stream: the smallest call
        dict(name="rotary_step_bf16", op="rotary", B=64, L=1, H=12, dh=64, rot=64, layout="half", scaling="none",
             far=1 << 20, dtype="bf16", grad=False),
        # a training step's rotation of half of each head, interleaved pairs
        dict(name="rotary_train_bf16", op="rotary", B=32, L=1024, H=12, dh=64, rot=32, layout="interleaved",
             scaling="none", far=0, dtype="bf16", grad=True),
        # the same step for one token: queries of 12 heads, keys of 4, normalised and rotated
        dict(name="norm_step_bf16", op="norm", B=64, L=1, Lk=1, H=12, Hk=4, dh=64, rot=64, layout="half",
             scaling="yarn", far=1 << 17, dtype="bf16", grad=False),
        # one training step of the small preset's heads on 8 frames of 196 tokens, with gradients of the weights
        dict(name="norm_train_bf16", op="norm", B=32, L=1568, Lk=1568, H=6, Hk=6, dh=64, rot=64, layout="half",
             scaling="none", far=0, dtype="bf16", grad=True),
        # float32, slots against the tokens of a frame and its class token: two odd lengths
        dict(name="norm_train_fp32", op="norm", B=32, L=31, Lk=197, H=8, Hk=8, dh=64, rot=48, layout="interleaved",
             scaling="linear", far=0, dtype="fp32", grad=True),
        # serving: one goal query for each clip against 8 frames of tokens, clips of different lengths, k and v
        # as they come out of one projection
        dict(name="cross_step_bf16", op="cross", B=64, Lq=1, Lk=1568, H=12, Hk=12, dh=64, keys="lens", fused=True,
             dtype="bf16", grad=False),
        # the same for one long stream with shared key heads: little to spread but the keys
        dict(name="cross_step_long_bf16", op="cross", B=1, Lq=1, Lk=100352, H=16, Hk=4, dh=128, keys="all",
             fused=False, dtype="bf16", grad=False),
        # 32 slots of every frame read its 196 tokens, float32 as the small preset runs without autocast
        dict(name="cross_slots_fp32", op="cross", B=64, Lq=32, Lk=196, H=6, Hk=6, dh=64, keys="all", fused=False,
             dtype="fp32", grad=False),
        # one training step of the same in bf16 over 16 clips of 16 frames
        dict(name="cross_slots_train_bf16", op="cross", B=256, Lq=32, Lk=196, H=6, Hk=6, dh=64, keys="all",
             fused=False, dtype="bf16", grad=True),
        # odd sizes with padded keys, one clip without any, heads of 80
        dict(name="cross_odd_train_fp16", op="cross", B=5, Lq=77, Lk=1003, H=8, Hk=2, dh=80, keys="mask",
             fused=False, dtype="fp16", grad=True),
        # long queries against a longer encoder, clips of different lengths
        dict(name="cross_long_bf16", op="cross", B=8, Lq=2048, Lk=4099, H=12, Hk=12, dh=64, keys="lens",
             fused=True, dtype="bf16", grad=False),
        # the largest: a training step with heads of 128 shared by groups of three
        dict(name="cross_train_bf16", op="cross", B=8, Lq=1024, Lk=2048, H=12, Hk=4, dh=128, keys="all",
             fused=False, dtype="bf16", grad=True),
    ]


# ------------------------------------------------------------------------------------------------ drawn cases

def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    """One more case: the operator, its sizes, types and options over the ranges of the listed ones."""
    op = rng.choice(("rotary", "norm", "cross", "cross", "cross"))
    dtype = rng.choice(("fp32", "bf16", "bf16", "fp16"))
    grad = rng.random() < 0.5
    if op != "cross":
        dh = rng.choice((32, 64, 64, 80, 96, 128, 192, 256))
        H = rng.randint(1, 16)
        L = 1 if rng.random() < 0.25 else _log(rng, 2, 4096)
        B = _log(rng, 1, max(1, min(256, int(2.0e7 / (L * H * dh)))))
        case = dict(op=op, B=B, L=L)
        if op == "norm":
            case.update(Lk=L if rng.random() < 0.6 else max(1, int(L * rng.uniform(0.2, 1.0))))
        case.update(H=H)
        if op == "norm":
            case.update(Hk=rng.choice([g for g in range(1, H + 1) if H % g == 0]))
        case.update(dh=dh, rot=rng.choice((dh, dh, dh // 2, dh // 4 // 2 * 2, dh - 2)),
                    layout=rng.choice(("half", "interleaved")), scaling=rng.choice(("none", "linear", "ntk", "yarn")),
                    far=rng.choice((0, 0, 1 << 12, 1 << 17, 1 << 20)), dtype=dtype, grad=grad)
        return case
    dh = rng.choice((32, 64, 64, 80, 96, 128, 128, 256))
    Hk = rng.randint(1, 12)
    H = Hk * rng.choice((1, 1, 1, 2, 3, 4))
    Lk = _log(rng, 1, 8192)
    Lq = 1 if rng.random() < 0.3 else _log(rng, 2, 2048)
    cost = Lq * Lk * H * dh * (3.5 if grad else 1.0) * (8.0 if dtype == "fp32" else 1.0)
    room = max(Lq * H, Lk * Hk) * dh
    B = _log(rng, 1, max(1, min(128, int(min(4.0e10 / cost, 5.0e7 / room)))))
    return dict(op=op, B=B, Lq=Lq, Lk=Lk, H=H, Hk=Hk, dh=dh, keys=rng.choice(("all", "lens", "mask")),
                fused=not grad and rng.random() < 0.3, dtype=dtype, grad=grad)


# ---------------------------------------------------------------------------------------------------- inputs

def _key_counts(case) -> list:
    """Live keys of each batch row; how they are spread over the rows changes with the seed, their sum does not."""
    B, Lk = case["B"], case["Lk"]
    if case["keys"] == "lens":      # from a quarter of the keys to all of them
        return [max(1, round(Lk * (0.25 + 0.75 * (i + 1) / B))) for i in range(B)]
    if case["keys"] == "mask":      # four in five; of four or more rows one has no key at all
        return [0 if B >= 4 and i == 0 else Lk - Lk // 5 for i in range(B)]
    return [Lk] * B


_SCALING = {"none": dict(), "linear": dict(scaling="linear", factor=4.0), "ntk": dict(scaling="ntk", factor=4.0),
            "yarn": dict(scaling="yarn", factor=8.0, original_length=4096)}


def _frequencies(rot: int, scaling: str):
    """Frequency of each pair in float64, and the factor on the rotated values."""
    base, n = 10000.0, rot // 2
    opt = _SCALING[scaling]
    i = torch.arange(n, dtype=torch.float64)
    if scaling == "ntk":
        base = base * opt["factor"] ** (rot / (rot - 2)) if rot > 2 else base
    f = base ** (-2.0 * i / rot)
    if scaling == "linear":
        f = f / opt["factor"]
    if scaling == "yarn":
        def pair_of(turns):        # the (real) pair index that makes this many turns over the original length
            return rot * math.log(opt["original_length"] / (2 * math.pi * turns)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), rot - 1)
        keep = 1.0 - ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        f = f * keep + f / opt["factor"] * (1.0 - keep)
        return f, 0.1 * math.log(opt["factor"]) + 1.0
    return f, 1.0


def _positions(case, L, g):
    if L == 1 or case["far"]:       # every row at its own place of its stream
        start = torch.randint(0, max(case["far"], 4096), (case["B"], 1), generator=g, device="cuda")
        return start + torch.arange(L, device="cuda")
    return torch.arange(L, device="cuda")


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    op, B, H, dh = case["op"], case["B"], case["H"], case["dh"]

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dt)

    st = dict(case=case)
    if op == "cross":
        Lq, Lk, Hk = case["Lq"], case["Lk"], case["Hk"]
        st["q"] = rand(B, Lq, H, dh)
        if case["fused"]:
            kv = rand(B, Lk, 2, Hk, dh)
            st["k"], st["v"] = kv[:, :, 0], kv[:, :, 1]
        else:
            st["k"], st["v"] = rand(B, Lk, Hk, dh), rand(B, Lk, Hk, dh)
        order = torch.randperm(B, generator=g, device="cuda")
        counts = torch.tensor(_key_counts(case), device="cuda")[order]
        st["lens"] = counts.to(torch.int32) if case["keys"] == "lens" else None
        st["mask"] = None
        if case["keys"] == "mask":
            rank = torch.rand(B, Lk, generator=g, device="cuda").argsort(1).argsort(1)
            st["mask"] = rank >= counts[:, None]              # True = not read
        if case["grad"]:
            st["gy"] = rand(B, Lq, H, dh)
            leaves = ("q", "k", "v")
    else:
        freq, amp = _frequencies(case["rot"], case["scaling"])
        st["freq"], st["amp"] = freq.cuda(), amp
        st["pos"] = _positions(case, case["L"], g)
        if own:
            from hclsm_amd.kernels import RotaryPlan
            st["plan"] = RotaryPlan(case["rot"], layout=case["layout"], **_SCALING[case["scaling"]])
        if op == "rotary":
            st["x"] = rand(B, case["L"], H, dh)
            leaves = ("x",)
            if case["grad"]:
                st["gy"] = rand(B, case["L"], H, dh)
        else:
            st["q"], st["k"] = rand(B, case["L"], H, dh), rand(B, case["Lk"], case["Hk"], dh)
            st["kpos"] = st["pos"] if case["Lk"] == case["L"] else _positions(case, case["Lk"], g)
            for name in ("wq", "wk"):
                st[name] = 1.0 + 0.2 * torch.randn(dh, generator=g, device="cuda")
            leaves = ("q", "k", "wq", "wk")
            if case["grad"]:
                st["gq"], st["gk"] = rand(B, case["L"], H, dh), rand(B, case["Lk"], case["Hk"], dh)
    if own and case["grad"]:
        for name in leaves:
            st[name].requires_grad_()
    return st


# ------------------------------------------------------------------------------------------------ plain form

def _cos_sin(pos, freq, amp):
    """cos and sin of every position and pair, (B or 1, L, 1, pairs): angles in float64, values in float32."""
    a = pos.reshape(-1, pos.shape[-1], 1, 1).double() * freq
    return (amp * torch.cos(a)).float(), (amp * torch.sin(a)).float()


def _rotate(x, cos, sin, rot, layout):
    """Float32 heads x rotated by the angles; sin negated turns back (the gradient)."""
    if layout == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((y, x[..., rot:]), -1) if rot < x.shape[-1] else y


def _plain_rotary(st):
    case = st["case"]
    cos, sin = _cos_sin(st["pos"], st["freq"], st["amp"])
    dt = st["x"].dtype
    y = _rotate(st["x"].float(), cos, sin, case["rot"], case["layout"]).to(dt)
    if not case["grad"]:
        return y
    return y, _rotate(st["gy"].float(), cos, -sin, case["rot"], case["layout"]).to(dt)


def _plain_norm(st):
    case = st["case"]
    outs, grads, wgrads = [], [], []
    for name, pos in (("q", "pos"), ("k", "kpos")):
        x, w = st[name], st["w" + name]
        cos, sin = _cos_sin(st[pos], st["freq"], st["amp"])
        xf = x.float()
        r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + _EPS)
        n = xf * r
        outs.append(_rotate(n * w, cos, sin, case["rot"], case["layout"]).to(x.dtype))
        if case["grad"]:
            d = _rotate(st["g" + name].float(), cos, -sin, case["rot"], case["layout"])
            dn = d * w
            grads.append((r * (dn - n * (dn * n).mean(-1, keepdim=True))).to(x.dtype))
            wgrads.append((d * n).sum((0, 1, 2)))
    return tuple(outs + grads + wgrads)


def _plain_cross(st):
    case = st["case"]
    q, k, v = st["q"], st["k"], st["v"]
    B, Lq, H, dh = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G, scale, dt = H // Hk, dh ** -0.5, q.dtype
    # the heads that share a key head are rows of one product: (B, Hk, Lq * G, dh)
    qf = q.float().reshape(B, Lq, Hk, G, dh).permute(0, 2, 1, 3, 4).reshape(B, Hk, Lq * G, dh)
    kf, vf = (t.float().permute(0, 2, 1, 3).contiguous() for t in (k, v))
    s = torch.matmul(qf, kf.transpose(-1, -2)) * scale
    dead = None
    if st["lens"] is not None:
        dead = torch.arange(Lk, device=q.device) >= st["lens"][:, None]
    elif st["mask"] is not None:
        dead = st["mask"]
    if dead is not None:
        s = s.masked_fill(dead[:, None, None, :], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)     # no key: a row of zeros
    o = torch.matmul(p, vf)

    def heads(t):
        return t.reshape(B, Hk, Lq, G, dh).permute(0, 2, 1, 3, 4).reshape(B, Lq, H, dh).to(dt)

    if not case["grad"]:
        return heads(o)
    gf = st["gy"].float().reshape(B, Lq, Hk, G, dh).permute(0, 2, 1, 3, 4).reshape(B, Hk, Lq * G, dh)
    dv = torch.matmul(p.transpose(-1, -2), gf)
    dp = torch.matmul(gf, vf.transpose(-1, -2))
    ds = p * (dp - (gf * o).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, kf)
    dk = torch.matmul(ds.transpose(-1, -2), qf)
    return (heads(o), heads(dq), dk.permute(0, 2, 1, 3).contiguous().to(dt),
            dv.permute(0, 2, 1, 3).contiguous().to(dt))


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    case = state["case"]
    if not own:
        return {"rotary": _plain_rotary, "norm": _plain_norm, "cross": _plain_cross}[case["op"]](state)
    from hclsm_amd.kernels import cross_attention, qk_norm_rotary, rotary_embedding
    if case["op"] == "rotary":
        y = rotary_embedding(state["x"], state["plan"], state["pos"])
        if not case["grad"]:
            return y
        return (y.detach(),) + torch.autograd.grad(y, (state["x"],), state["gy"])
    if case["op"] == "norm":
        y = qk_norm_rotary(state["q"], state["k"], state["wq"], state["wk"], state["plan"], state["pos"],
                           state["kpos"], eps=_EPS)
        if not case["grad"]:
            return y
        leaves = tuple(state[n] for n in ("q", "k", "wq", "wk"))
        return tuple(t.detach() for t in y) + torch.autograd.grad(y, leaves, (state["gq"], state["gk"]))
    y = cross_attention(state["q"], state["k"], state["v"], key_lens=state["lens"], key_padding_mask=state["mask"])
    if not case["grad"]:
        return y
    return (y.detach(),) + torch.autograd.grad(y, tuple(state[n] for n in ("q", "k", "v")), state["gy"])


def work(case) -> dict:
    """Each input read once, each output written once; products of the definition (a multiply and an add are two)."""
    e, B, H, dh = _SIZE[case["dtype"]], case["B"], case["H"], case["dh"]
    grad = case["grad"]
    if case["op"] == "rotary":
        n = B * case["L"] * H * dh
        return dict(bytes=(4 if grad else 2) * n * e, flops=(6 if grad else 3) * n * case["rot"] // dh)
    if case["op"] == "norm":
        n = B * dh * (case["L"] * H + case["Lk"] * case["Hk"])
        return dict(bytes=(4 if grad else 2) * n * e + (4 if grad else 2) * dh * 4, flops=(20 if grad else 7) * n)
    live = sum(_key_counts(case))
    nq, nk = B * case["Lq"] * H * dh, live * case["Hk"] * dh
    full = B * case["Lk"] * case["Hk"] * dh        # gradients are written for the keys that are not read too
    b = (2 * nq + 2 * nk) * e + ((2 * nq + 2 * full) * e if grad else 0)
    return dict(bytes=b, flops=live * case["Lq"] * H * dh * (14 if grad else 4))


# --------------------------------------------------------------------------------------- the definition in float64

def _turn(x, pos, freq, amp, rot, layout):
    """Each pair of a head as one complex number, times amp * exp(i * position * frequency)."""
    first = list(range(rot // 2)) if layout == "half" else list(range(0, rot, 2))
    second = list(range(rot // 2, rot)) if layout == "half" else list(range(1, rot, 2))
    ang = pos.double()[..., None] * freq
    if ang.dim() == 2:
        ang = ang[None]
    z = torch.complex(x[..., first], x[..., second]) * (amp * torch.polar(torch.ones_like(ang), ang))[:, :, None, :]
    y = torch.cat((z.real, z.imag, x[..., rot:]), -1)
    back = torch.empty(x.shape[-1], dtype=torch.long, device=x.device)
    back[torch.tensor(first + second + list(range(rot, x.shape[-1])), device=x.device)] = \
        torch.arange(x.shape[-1], device=x.device)
    return y[..., back]


def _laid_out_alike(outs, grads):
    res = tuple(o.detach() for o in outs) + tuple(grads)
    return res[0] if len(res) == 1 else res


def exact(case, seed):
    st = prepare(case, seed)
    op, grad = case["op"], case["grad"]
    if op == "cross":
        # one batch row and key head at a time: the scores of a whole long case do not fit in float64
        G, outs = case["H"] // case["Hk"], None
        q, k, v = (st[n].detach() for n in ("q", "k", "v"))
        names = ("o", "q", "k", "v") if grad else ("o",)
        outs = {n: torch.zeros((k if n in "kv" else q).shape, dtype=torch.float64, device="cuda") for n in names}
        for b in range(case["B"]):
            if st["lens"] is not None:
                live = torch.arange(case["Lk"], device="cuda")[:int(st["lens"][b])]
            elif st["mask"] is not None:
                live = torch.nonzero(~st["mask"][b])[:, 0]
            else:
                live = torch.arange(case["Lk"], device="cuda")
            if live.numel() == 0:
                continue
            qb = q[b].double().requires_grad_(grad)
            kb, vb = (t[b, live].double().requires_grad_(grad) for t in (k, v))
            ys = []
            for h in range(case["H"]):
                w = torch.softmax(qb[:, h] @ kb[:, h // G].t() / math.sqrt(case["dh"]), -1)
                ys.append(w @ vb[:, h // G])
            y = torch.stack(ys, 1)
            outs["o"][b] = y.detach()
            if grad:
                gq, gk, gv = torch.autograd.grad(y, (qb, kb, vb), st["gy"][b].double())
                outs["q"][b] = gq
                outs["k"][b, live] = gk
                outs["v"][b, live] = gv
        return outs["o"] if not grad else tuple(outs[n] for n in names)
    freq, amp = _frequencies(case["rot"], case["scaling"])
    freq = freq.cuda()
    if op == "rotary":
        x = st["x"].detach().double().requires_grad_(grad)
        y = _turn(x, st["pos"], freq, amp, case["rot"], case["layout"])
        return _laid_out_alike((y,), torch.autograd.grad(y, (x,), st["gy"].double()) if grad else ())
    leaves = [st[n].detach().double().requires_grad_(grad) for n in ("q", "k", "wq", "wk")]
    ys = []
    for x, w, pos in ((leaves[0], leaves[2], st["pos"]), (leaves[1], leaves[3], st["kpos"])):
        rms = torch.sqrt((x ** 2).sum(-1, keepdim=True) / case["dh"] + _EPS)
        ys.append(_turn(x / rms * w, pos, freq, amp, case["rot"], case["layout"]))
    grads = torch.autograd.grad(ys, leaves, (st["gq"].double(), st["gk"].double())) if grad else ()
    return _laid_out_alike(ys, grads)
