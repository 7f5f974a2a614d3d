"""Linear attention with a decay per head and norms with the residual's addition as measured cases.

    mix      linear_attention: prompts in chunks, with the state before and behind them, or a training step's gradients
    step     linear_attention_step: one token of many streams, their states updated in place
    norm     residual_rms_norm: the residual's addition and the root-mean-square norm, alone or with gradients
    fp8      residual_rms_norm_fp8: the same with its output in 8 bits and scales by row or by group of columns

With ``own`` false, ``run`` computes the plain form: elementary torch operations in float32 (powers of the decay in
float64), rounded once at the end.  With ``own`` true it makes a user's calls of ``hclsm_amd.kernels``.  ``exact``
restates each operator in float64 and takes gradients by differentiating that statement.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
_EPS = 1e-6
_CHUNK = 64


def listed() -> list:
    return [
        # serving, one new token for each of 16 clips: the smallest call
        dict(name="step_bf16", op="step", B=16, pool=16, H=12, Hk=12, dk=64, dv=64, decay="slow", dtype="bf16"),
        # serving at full load: 256 streams out of a pool of 320 states, heads of 128
        dict(name="step_pool_bf16", op="step", B=256, pool=320, H=16, Hk=16, dk=128, dv=128, decay="slow",
             dtype="bf16"),
        # the prompt of one long stream, 32 x 8 frames of 196 tokens: little to spread but time
        dict(name="mix_stream_bf16", op="mix", B=1, L=50176, H=12, Hk=12, dk=64, dv=64, decay="slow", lens=False,
             state=True, dtype="bf16", grad=False),
        # prompts of different lengths that go on from kept states, key heads shared by four, two odd sizes
        dict(name="mix_ragged_fp16", op="mix", B=7, L=1003, H=8, Hk=2, dk=64, dv=80, decay="mixed", lens=True,
             state=True, dtype="fp16", grad=False),
        # one training step of 12 heads of 64 over 32 clips
        dict(name="mix_train_bf16", op="mix", B=32, L=1024, H=12, Hk=12, dk=64, dv=64, decay="slow", lens=False,
             state=False, dtype="bf16", grad=True),
        # float32 over a frame's tokens and its class token, gradients of the state too
        dict(name="mix_train_fp32", op="mix", B=16, L=197, H=6, Hk=6, dk=48, dv=96, decay="mixed", lens=False,
             state=True, dtype="fp32", grad=True),
        # the largest: a training step with heads of 128 over long clips
        dict(name="mix_train_large_bf16", op="mix", B=8, L=4096, H=16, Hk=16, dk=128, dv=128, decay="slow",
             lens=False, state=False, dtype="bf16", grad=True),
        # one token of 64 clips at the base width
        dict(name="norm_step_bf16", op="norm", rows=64, D=768, stream="same", dtype="bf16", grad=False),
        # a training step of the small width on 32 x 8 frames of 196 tokens
        dict(name="norm_train_bf16", op="norm", rows=50176, D=384, stream="same", dtype="bf16", grad=True),
        # odd rows and columns, half precision on a float32 stream
        dict(name="norm_odd_fp16", op="norm", rows=8027, D=1001, stream="fp32", dtype="fp16", grad=True),
        # one token of 32 clips into 8 bits
        dict(name="fp8_step_bf16", op="fp8", rows=32, D=768, stream="same", group=0, dtype="bf16"),
        # a long prompt into 8 bits with a scale for each 128 columns
        dict(name="fp8_prompt_bf16", op="fp8", rows=32768, D=4096, stream="same", group=128, dtype="bf16"),
    ]


# ------------------------------------------------------------------------------------------------ drawn cases

def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    """One more case: the operator, its sizes, types and options over the ranges of the listed ones."""
    op = rng.choice(("mix", "mix", "mix", "step", "norm", "fp8"))
    dtype = rng.choice(("fp32", "bf16", "bf16", "fp16"))
    if op in ("norm", "fp8"):
        D = _log(rng, 8, 8192)
        group = 0
        if op == "fp8" and rng.random() < 0.5:
            group = rng.choice((32, 64, 128))
            D = max(group, D // group * group)
        rows = _log(rng, 1, max(1, min(65536, int(1.3e8 / D))))
        case = dict(op=op, rows=rows, D=D, stream=rng.choice(("same", "same", "fp32", "none")))
        if op == "fp8":
            return dict(case, group=group, dtype=dtype)
        return dict(case, dtype=dtype, grad=rng.random() < 0.5)
    dk, dv = rng.choice((32, 48, 64, 64, 96, 128, 128, 256)), rng.choice((32, 64, 64, 80, 96, 128, 128, 256))
    Hk = rng.randint(1, 16)
    H = Hk * rng.choice((1, 1, 1, 1, 2, 4))
    decay = rng.choice(("slow", "slow", "mixed"))
    if op == "step":
        B = _log(rng, 1, max(1, min(256, int(6.7e7 / (H * dk * dv)))))
        return dict(op=op, B=B, pool=B + rng.choice((0, 0, 1, B // 4 + 1)), H=H, Hk=Hk, dk=dk, dv=dv, decay=decay,
                    dtype=dtype)
    grad = rng.random() < 0.5
    L = _log(rng, 1, 16384)
    most = 6.7e7 if grad else 1.0e8
    B = _log(rng, 1, max(1, min(64, int(most * (0.5 if dtype == "fp32" else 1.0) / (L * H * (dk + dv) / 2)),
                                int(8.0e9 / (max(L, 64) * H * dk * dv)))))
    return dict(op=op, B=B, L=L, H=H, Hk=Hk, dk=dk, dv=dv, decay=decay, lens=rng.random() < 0.3,
                state=rng.random() < 0.5, dtype=dtype, grad=grad)


# ---------------------------------------------------------------------------------------------------- inputs

def _log_decay(case):
    """(H,) float32.  slow: memories from 32 to 4096 tokens; mixed: those, none at all, and a sum without decay."""
    H = case["H"]
    i = torch.arange(H, dtype=torch.float64) / max(H - 1, 1)
    g = torch.log1p(-(2.0 ** (-5.0 - 7.0 * i)))
    if case["decay"] == "mixed":
        g[0] = 0.0
        if H > 1:
            g[1] = -2.5
    return g.float()


def _live(case) -> list:
    """Live tokens of each row: from a quarter of them to all, and of four or more rows one has none."""
    B, L = case["B"], case["L"]
    if not case["lens"]:
        return [L] * B
    return [0 if B >= 4 and i == 0 else max(1, round(L * (0.25 + 0.75 * (i + 1) / B))) for i in range(B)]


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    op = case["op"]

    def rand(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    st = dict(case=case)
    leaves = ()
    if op in ("norm", "fp8"):
        rows, D = case["rows"], case["D"]
        st["x"] = rand(rows, D)
        sdt = torch.float32 if case["stream"] == "fp32" else dt
        st["r"] = None if case["stream"] == "none" else (2.0 * rand(rows, D, dtype=torch.float32)).to(sdt)
        st["w"] = 1.0 + 0.2 * torch.randn(D, generator=g, device="cuda")
        if case.get("grad"):
            st["gy"] = rand(rows, D)
            st["gh"] = rand(rows, D, dtype=sdt if st["r"] is not None else dt)
            leaves = ("x", "r", "w")
    else:
        B, H, Hk, dk, dv = (case[n] for n in ("B", "H", "Hk", "dk", "dv"))
        st["g"] = _log_decay(case).cuda()
        if op == "step":
            st["q"], st["k"], st["v"] = rand(B, H, dk), rand(B, Hk, dk), rand(B, Hk, dv)
            st["s"] = 4.0 * rand(case["pool"], H, dk, dv, dtype=torch.float32)
            st["rows"] = None
            if case["pool"] != B:
                st["rows"] = torch.randperm(case["pool"], generator=g, device="cuda")[:B].to(torch.int32)
        else:
            L = case["L"]
            st["q"], st["k"], st["v"] = rand(B, L, H, dk), rand(B, L, Hk, dk), rand(B, L, Hk, dv)
            st["s"] = 4.0 * rand(B, H, dk, dv, dtype=torch.float32) if case["state"] else None
            order = torch.randperm(B, generator=g, device="cuda")
            st["lens"] = torch.tensor(_live(case), device="cuda")[order].to(torch.int32) if case["lens"] else None
            if case["grad"]:
                st["go"] = rand(B, L, H, dv)
                st["gs"] = rand(B, H, dk, dv, dtype=torch.float32) if case["state"] else None
                leaves = ("q", "k", "v", "s")
    for name in leaves:
        if st[name] is not None:
            st[name].requires_grad_()
    st["leaves"] = tuple(n for n in leaves if st[n] is not None)
    return st


# ------------------------------------------------------------------------------------------------ plain form

def _powers(g, n):
    """(H, n + 1): the decay's powers 0 .. n, formed in float64."""
    return torch.exp(g.double()[:, None] * torch.arange(n + 1, device=g.device, dtype=torch.float64))


def _mix(a, b, x, s, g, live, shift, cp, ci, cu):
    """y_t = cp sum_{s <= t} d^(t-s) (a_t b_s) x_s + ci d^(t+1-shift) a_t S, and cu sum_s d^(n-1-s+shift) b_s x_s' + d^n S,
    of (B, H, L, .) tensors in float32; live (B,): the tokens behind it are zeros already, and count for no power.

    Chunks of a fixed size, all at once: products inside them, their sums b x', and what reaches a chunk from the
    earlier ones by the matrix of the decay's powers between chunks."""
    B, H, L, da = a.shape
    dx, C = x.shape[-1], _CHUNK
    n = -(-max(L, 1) // C)
    pad = n * C - L
    a, b, x = (torch.nn.functional.pad(t, (0, 0, 0, pad)).reshape(B, H, n, C, t.shape[-1]) for t in (a, b, x))
    pw = _powers(g, C)
    i = torch.arange(C, device=g.device)
    inside = torch.where(i[:, None] >= i[None, :], pw[:, (i[:, None] - i[None, :]).clamp(min=0)], 0.0).float()
    p = torch.matmul(a, b.transpose(-1, -2)) * (cp * inside)[None, :, None]
    y = torch.matmul(p, x)
    u = torch.matmul((b * pw[:, C - 1 - i].float()[None, :, None, :, None]).transpose(-1, -2), x)
    u = u.reshape(B, H, n, da * dx)
    j = torch.arange(n, device=g.device)
    gap = (j[:, None] - 1 - j[None, :]).clamp(min=0)
    across = torch.where(j[:, None] > j[None, :], torch.exp(g.double()[:, None, None] * (C * gap)), 0.0).float()
    start = torch.matmul(across[None], u) * cu              # sums in front of each chunk, without the shift
    if s is not None:
        first = torch.exp(g.double()[:, None] * (C * j)).float()
        start = start * pw[:, shift].float()[None, :, None, None]
        start = start + first[None, :, :, None] * s.reshape(B, H, 1, da * dx)
    elif shift:
        start = start * pw[:, shift].float()[None, :, None, None]
    start = start.reshape(B, H, n, da, dx)
    y = y + ci * torch.matmul(a * pw[:, i + 1 - shift].float()[None, :, None, :, None], start)
    y = y.reshape(B, H, n * C, dx)[:, :, :L]
    # the state behind the last live token: the chunk it lies in, with the powers from that token on
    c = ((live - 1).clamp(min=0) // C).long()
    m = (live - c * C).clamp(min=0)                         # live tokens of that chunk
    rest = (m[:, None] - 1 - i[None, :])
    w = torch.exp(g.double()[None, :, None] * (rest + shift).clamp(min=0)[:, None, :])
    w = torch.where(rest[:, None, :] >= 0, w, 0.0).float()
    at = c[:, None, None, None, None]
    bl = b.gather(2, at.expand(B, H, 1, C, da))[:, :, 0]
    xl = x.gather(2, at.expand(B, H, 1, C, dx))[:, :, 0]
    sl = start.gather(2, at.expand(B, H, 1, da, dx))[:, :, 0]
    end = cu * torch.matmul((bl * w[..., None]).transpose(-1, -2), xl)
    end = end + torch.exp(g.double()[None, :] * m[:, None]).float()[..., None, None] * sl
    return y, end


def _plain_mix(st):
    case = st["case"]
    H, Hk, L, B = case["H"], case["Hk"], case["L"], case["B"]
    c, dt, G = case["dk"] ** -0.5, st["q"].dtype, H // Hk
    live = st["lens"].long() if st["lens"] is not None else torch.full((B,), L, device="cuda")
    on = (torch.arange(L, device="cuda") < live[:, None])[:, None, :, None]

    def heads(t):
        t = t.float().permute(0, 2, 1, 3)
        return torch.where(on, t.repeat_interleave(H // t.shape[1], 1), 0.0)

    def rows(t, dtype=dt):
        return t.permute(0, 2, 1, 3).to(dtype).contiguous()

    q, k, v, s = heads(st["q"]), heads(st["k"]), heads(st["v"]), st["s"]
    y, end = _mix(q, k, v, s, st["g"], live, 0, c, c, 1.0)
    out = (rows(torch.where(on, y, 0.0)),) + ((end,) if case["state"] else ())
    if not case["grad"]:
        return out if case["state"] else out[0]
    do = heads(st["go"])
    # backwards in time: token t of a row with n live ones stands at n - 1 - t
    back = (live[:, None] - 1 - torch.arange(L, device="cuda"))
    turn = torch.where(back >= 0, back, torch.arange(L, device="cuda"))[:, None, :, None]
    rev = lambda t: t.gather(2, turn.expand(t.shape))  # noqa: E731
    tr = lambda t: None if t is None else t.transpose(-1, -2).contiguous()  # noqa: E731
    dq, _ = _mix(do, v, k, tr(s), st["g"], live, 0, c, c, 1.0)
    rq, rk, rv, rdo = rev(q), rev(k), rev(v), rev(do)
    dv, ds = _mix(rk, rq, rdo, st["gs"], st["g"], live, 1, c, 1.0, c)
    dk, _ = _mix(rv, rdo, rq, tr(st["gs"]), st["g"], live, 1, c, 1.0, c)
    dk, dv = (torch.where(on, rev(t), 0.0).reshape(B, Hk, G, L, t.shape[-1]).sum(2) for t in (dk, dv))
    grads = (rows(torch.where(on, dq, 0.0)), rows(dk), rows(dv)) + ((ds,) if case["state"] else ())
    return out + grads


def _plain_step(st):
    case = st["case"]
    G = case["H"] // case["Hk"]
    q, k, v = (st[n].float() for n in ("q", "k", "v"))
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    old = st["s"] if st["rows"] is None else st["s"][st["rows"].long()]
    new = old * torch.exp(st["g"].double()).float()[:, None, None] + k[..., :, None] * v[..., None, :]
    if st["rows"] is None:
        st["s"].copy_(new)
    else:
        st["s"][st["rows"].long()] = new
    y = (q[..., :, None] * new).sum(-2) * case["dk"] ** -0.5
    return y.to(st["q"].dtype), st["s"]


def _plain_norm(st):
    case = st["case"]
    x, r, w = st["x"], st["r"], st["w"]
    h = x if r is None else (x.float() + r.float()).to(r.dtype)      # the stream, as the next layer reads it
    hf = h.float()
    inv = torch.rsqrt((hf * hf).mean(-1, keepdim=True) + _EPS)
    n = hf * inv
    y = n * w
    if case["op"] == "fp8":
        D, group = case["D"], case["group"] or case["D"]
        yg = y.reshape(-1, D // group, group)
        scale = yg.abs().amax(-1).clamp(min=2.0 ** -100) / 448.0
        y8 = (yg / scale[..., None]).to(torch.float8_e4m3fn).reshape(y.shape)
        return (y8, scale) + (() if r is None else (h,))
    out = (y.to(x.dtype),) + (() if r is None else (h,))
    if not case["grad"]:
        return out
    gy = st["gy"].float()
    gn = gy * w
    dh = inv * (gn - n * (gn * n).mean(-1, keepdim=True)) + st["gh"].float()
    grads = (dh.to(x.dtype),) + (() if r is None else (dh.to(r.dtype),)) + ((gy * n).sum(0),)
    return out + grads


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return {"mix": _plain_mix, "step": _plain_step, "norm": _plain_norm, "fp8": _plain_norm}[case["op"]](state)
    from hclsm_amd.kernels import linear_attention, linear_attention_step, residual_rms_norm, residual_rms_norm_fp8
    leaves = tuple(state[n] for n in state["leaves"])
    if case["op"] == "step":
        y = linear_attention_step(state["q"], state["k"], state["v"], state["g"], state["s"], rows=state["rows"])
        return y, state["s"]
    if case["op"] == "mix":
        y = linear_attention(state["q"], state["k"], state["v"], state["g"], initial_state=state["s"],
                             seq_lens=state["lens"], return_state=case["state"])
        if not case["grad"]:
            return y
        y = y if case["state"] else (y,)
        gs = (state["go"], state["gs"]) if case["state"] else (state["go"],)
        return tuple(t.detach() for t in y) + torch.autograd.grad(y, leaves, gs)
    if case["op"] == "fp8":
        y8, scale, h = residual_rms_norm_fp8(state["x"], state["r"], state["w"], eps=_EPS, group=case["group"] or None)
        return (y8, scale) if state["r"] is None else (y8, scale, h)
    y, h = residual_rms_norm(state["x"], state["r"], state["w"], eps=_EPS)
    out = (y,) if state["r"] is None else (y, h)
    if not case["grad"]:
        return out
    return tuple(t.detach() for t in out) + torch.autograd.grad((y, h), leaves, (state["gy"], state["gh"]))


def work(case) -> dict:
    """Each input read once, each output written once; products of the definition (a multiply and an add are two), in the
    cheaper of the recurrent form and the one by pairs of tokens."""
    e = _SIZE[case["dtype"]]
    if case["op"] in ("norm", "fp8"):
        n = case["rows"] * case["D"]
        es = {"same": e, "fp32": 4, "none": 0}[case["stream"]]
        if case["op"] == "fp8":
            return dict(bytes=n * (e + 2 * es + 1) + n // (case["group"] or case["D"]) * 4 + case["D"] * 4, flops=7 * n)
        b = n * (2 * e + 2 * es) + case["D"] * 4
        if case["grad"]:        # the stream and both gradients of outputs read, those of the inputs written
            b += n * ((es or e) + e + (es or e) + e + (es if es not in (0, e) else 0)) + case["D"] * 8
        return dict(bytes=b, flops=(16 if case["grad"] else 5) * n)
    B, H, Hk, dk, dv = (case[n] for n in ("B", "H", "Hk", "dk", "dv"))
    if case["op"] == "step":
        return dict(bytes=8 * B * H * dk * dv + e * B * (H * (dk + dv) + Hk * (dk + dv)), flops=5 * B * H * dk * dv)
    live = _live(case)
    t, full = sum(live), B * case["L"]
    nq, nk, no = H * dk, Hk * (dk + dv), H * dv
    b = e * (t * (nq + nk) + full * no)
    if case["state"]:
        b += 8 * B * H * dk * dv
    if case["grad"]:
        b += e * (t * (nq + nk + no) + full * (nq + nk)) + (8 * B * H * dk * dv if case["state"] else 0)
    pairs = sum(n * (n + 1) // 2 for n in live)
    f = H * min(4 * t * dk * dv, pairs * 2 * (dk + dv))
    return dict(bytes=b, flops=f * (7 if case["grad"] else 2) // 2)


# --------------------------------------------------------------------------------------- the definition in float64

def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "fp8"):
        dt = st["x"].dtype
        x = st["x"].detach().double().requires_grad_()
        r = None if st["r"] is None else st["r"].detach().double().requires_grad_()
        w = st["w"].detach().double().requires_grad_()
        h = x if r is None else x + r
        if r is not None and st["r"].dtype != torch.float32:       # the stream's own values
            h = h + (h.detach().to(dt).double() - h.detach())
        y = h / torch.sqrt((h ** 2).sum(-1, keepdim=True) / case["D"] + _EPS) * w
        if op == "fp8":
            top = y.detach().reshape(case["rows"], -1, case["group"] or case["D"]).abs().amax(-1, keepdim=True)
            scale = torch.clamp(top, min=2.0 ** -100) / 448
            y8 = (y.detach().reshape(case["rows"], -1, case["group"] or case["D"]) / scale).reshape(y.shape)
            return (y8, scale[..., 0]) + (() if r is None else (h.detach(),))
        out = (y,) if r is None else (y, h)
        if not case["grad"]:
            return tuple(t.detach() for t in out)
        ins = (x, w) if r is None else (x, r, w)
        grads = torch.autograd.grad((y, h), ins, (st["gy"].double(), st["gh"].double()))
        return tuple(t.detach() for t in out) + grads
    G, c = case["H"] // case["Hk"], 1.0 / math.sqrt(case["dk"])
    a = torch.exp(st["g"].double())
    if op == "step":
        rows = torch.arange(case["B"], device="cuda") if st["rows"] is None else st["rows"].long()
        s, k, v = st["s"].double(), st["k"].double(), st["v"].double()
        y = torch.empty(case["B"], case["H"], case["dv"], dtype=torch.float64, device="cuda")
        for h in range(case["H"]):
            new = a[h] * s[rows, h] + torch.einsum("bi,bj->bij", k[:, h // G], v[:, h // G])
            s[rows, h] = new
            y[:, h] = c * torch.einsum("bi,bij->bj", st["q"][:, h].double(), new)
        return y, s
    B, L, H, dk, dv = (case[n] for n in ("B", "L", "H", "dk", "dv"))
    if B * H * L * L * (dk + dv) * (7 if case["grad"] else 2) > 2.0e14:
        return None
    q, k, v = (st[n].detach() for n in ("q", "k", "v"))
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device="cuda")  # noqa: E731
    s0 = None if st["s"] is None else st["s"].detach()
    outs = [torch.zeros(B, L, H, dv, dtype=torch.float64, device="cuda")] + ([z(s0)] if case["state"] else [])
    grads = [z(q), z(k), z(v)] + ([z(s0)] if case["state"] else []) if case["grad"] else []
    live = st["lens"].tolist() if st["lens"] is not None else [L] * B
    for b, n in enumerate(live):
        t = torch.arange(n, device="cuda", dtype=torch.float64)
        for h in range(H):
            ins = [q[b, :n, h].double(), k[b, :n, h // G].double(), v[b, :n, h // G].double()]
            ins += [s0[b, h].double()] if case["state"] else []
            ins = [i.requires_grad_(case["grad"]) for i in ins]
            age = t[:, None] - t[None, :]
            w = torch.where(age >= 0, torch.exp(st["g"][h].double() * age.clamp(min=0)), 0.0)
            y = c * ((w * (ins[0] @ ins[1].t())) @ ins[2])
            res = [y]
            if case["state"]:
                y = y + c * a[h] ** (t + 1)[:, None] * (ins[0] @ ins[3])
                res = [y, a[h] ** n * ins[3] + (ins[1] * (a[h] ** (n - 1 - t))[:, None]).t() @ ins[2]]
            outs[0][b, :n, h] = y.detach()
            if case["state"]:
                outs[1][b, h] = res[1].detach()
            if case["grad"]:
                up = [st["go"][b, :n, h].double()] + ([st["gs"][b, h].double()] if case["state"] else [])
                got = torch.autograd.grad(res, ins, up)
                grads[0][b, :n, h] = got[0]
                grads[1][b, :n, h // G] += got[1]
                grads[2][b, :n, h // G] += got[2]
                if case["state"]:
                    grads[3][b, h] = got[3]
    res = tuple(outs + grads)
    return res if len(res) > 1 else res[0]
