"""Position rotation of heads, alone and behind the norm of queries and keys (libhclsm_amd.so: hclsm_norm_rotary_*).

    plan = RotaryPlan(64)                                      # once per model
    y = rotary_embedding(x, plan, positions)                   # x (B, L, H, dh)
    q, k = qk_norm_rotary(q, k, q_weight, k_weight, plan, positions, key_positions)

Every head is turned in pairs: pair i of the plan's first ``rot_dim`` elements by position * frequency_i.  The norm is
the root mean square over a head's dh elements, in the same pass.  Both are differentiable (gradients of x, q, k and
the weights), with float32 arithmetic between the load and the one rounding at the store, and angles in float64; their
sines and cosines are float32 values within 1.4 times 2^-24.

x, q and k are (B, L, H, dh) tensors on the GPU (bfloat16, float16 or float32) of any strides whose last dimension is
contiguous (others are copied), 1 <= dh <= 256.  positions: int32 or int64, (L,) or (B, L); None counts from 0.  Outputs
are contiguous and new.  The reference rotates the heads of its vision encoder (perception/vision_encoder.py:171-259).
"""

from __future__ import annotations

import math

import torch

from hclsm_amd import _lib
from hclsm_amd.kernels._common import on_device, once, require_gpu
from hclsm_amd.kernels.ssm_scan_kernel import _no_node

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_LAYOUTS = {"half": _lib.ROTARY_HALF, "interleaved": _lib.ROTARY_INTERLEAVED}
MAX_HEAD_DIM = 256


class RotaryPlan:
    """Frequencies of a rotation, laid out once.

    rot_dim: elements of each head that are turned (even; the rest passes through).
    layout: "half" pairs elements i and i + rot_dim / 2, "interleaved" elements 2i and 2i + 1.
    base: frequency of pair i is base ** (-2 i / rot_dim).
    scaling, for contexts ``factor`` times as long as the model was trained on:
        "linear": every frequency divided by factor (positions interpolated);
        "ntk":    base * factor ** (rot_dim / (rot_dim - 2)), which leaves the fastest pair as it is and slows the
                  slowest one by factor;
        "yarn":   pairs that turn more than beta_fast times over original_length positions are kept, those that turn
                  less than beta_slow times are divided by factor, a linear ramp over the pair index between, and
                  the rotated values multiplied by 0.1 ln(factor) + 1 (Peng et al. 2023, "YaRN").
    amplitude: factor on the rotated values, in place of the scaling's own.
    inv_freq: (rot_dim / 2,) frequencies of the caller's, in place of base and scaling.

    ``inv_freq`` (float64, CPU) and ``amplitude`` hold the result.
    """

    def __init__(self, rot_dim: int, *, layout: str = "half", base: float = 10000.0, scaling: str | None = None,
                 factor: float = 1.0, original_length: int | None = None, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, amplitude: float | None = None, inv_freq: torch.Tensor | None = None,
                 device="cuda"):
        if rot_dim < 2 or rot_dim % 2 or rot_dim > MAX_HEAD_DIM:
            raise ValueError(f"rot_dim must be even and in [2, {MAX_HEAD_DIM}], got {rot_dim}")
        if layout not in _LAYOUTS:
            raise ValueError(f"layout must be one of {sorted(_LAYOUTS)}, got {layout!r}")
        if not base > 1 or not factor > 0:
            raise ValueError(f"base must be > 1 and factor > 0, got {base} and {factor}")
        n = rot_dim // 2
        amp = 1.0
        if inv_freq is not None:
            if scaling is not None:
                raise ValueError("give either inv_freq or a scaling")
            f = inv_freq.detach().to("cpu", torch.float64).contiguous()
            if f.shape != (n,) or not torch.isfinite(f).all():
                raise ValueError(f"inv_freq must be {n} finite frequencies, got shape {tuple(f.shape)}")
        else:
            b = base
            if scaling == "ntk" and rot_dim > 2:
                b = base * factor ** (rot_dim / (rot_dim - 2))
            i = torch.arange(n, dtype=torch.float64)
            f = b ** (-2.0 * i / rot_dim)
            if scaling == "linear":
                f = f / factor
            elif scaling == "yarn":
                if not original_length or original_length < 1:
                    raise ValueError("the yarn scaling needs original_length")
                if not beta_fast > beta_slow > 0:
                    raise ValueError(f"beta_fast must exceed beta_slow > 0, got {beta_fast} and {beta_slow}")
                pair = lambda turns: (rot_dim * math.log(original_length / (2 * math.pi * turns))
                                      / (2 * math.log(base)))
                lo, hi = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), rot_dim - 1)
                slow = ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
                f = f * (1.0 - slow) + f / factor * slow
                amp = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
            elif scaling not in (None, "ntk"):
                raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
        self.rot_dim, self.layout = int(rot_dim), layout
        self.inv_freq = f
        self.amplitude = float(amp if amplitude is None else amplitude)
        turns = f / (2 * math.pi)
        self._turns = torch.stack((turns, -turns)).to(device)     # forward, and turning back
        self._code = _LAYOUTS[layout]

    @property
    def device(self) -> torch.device:
        return self._turns.device


class _RawPlan:
    """What the kernels need of a plan, from tensors (the torch.library ops)."""

    def __init__(self, turns, rot_dim, code, amplitude):
        self._turns, self.rot_dim, self._code, self.amplitude = turns, rot_dim, code, amplitude

    @classmethod
    def of(cls, fn, turns, rot_dim, layout, amplitude, x):
        if rot_dim == 0:
            return None
        if rot_dim < 0 or rot_dim % 2 or rot_dim > x.shape[3] or layout not in _LAYOUTS.values():
            raise ValueError(f"{fn}: rot_dim must be even and at most {x.shape[3]}, layout 0 or 1, got {rot_dim} and {layout}")
        if turns is None or turns.dtype != torch.float64 or turns.shape != (rot_dim // 2,) or not turns.is_contiguous():
            raise ValueError(f"{fn}: turns must be {rot_dim // 2} contiguous float64 values")
        return cls(turns, rot_dim, layout, amplitude)


def _check_weight(fn, name, w, x):
    if w is not None and (w.shape != (x.shape[3],) or w.dtype not in _FLOATS or not w.is_contiguous()):
        raise ValueError(f"{fn}: {name} must be a contiguous float tensor of {x.shape[3]} elements, got "
                         f"{w.dtype} {tuple(w.shape)}")


def _check_heads(fn, name, x):
    if x.dim() != 4:
        raise ValueError(f"{fn}: {name} must be (B, L, H, dh), got shape {tuple(x.shape)}")
    if x.dtype not in _FLOATS:
        raise TypeError(f"{fn}: {name} must be bfloat16, float16 or float32, got {x.dtype}")
    if not 1 <= x.shape[3] <= MAX_HEAD_DIM:
        raise ValueError(f"{fn}: heads of 1 to {MAX_HEAD_DIM} elements, got {x.shape[3]}")


def _check_plan(fn, plan, dh):
    if plan is None:
        return
    if not isinstance(plan, RotaryPlan):
        raise TypeError(f"{fn}: plan must be a RotaryPlan, got {type(plan).__name__}")
    if plan.rot_dim > dh:
        raise ValueError(f"{fn}: the plan turns {plan.rot_dim} elements of heads of {dh}")


def _check_positions(fn, name, pos, x):
    if pos is None:
        return
    if pos.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{fn}: {name} must be int32 or int64, got {pos.dtype}")
    B, L = x.shape[:2]
    if tuple(pos.shape) not in ((L,), (B, L)):
        raise ValueError(f"{fn}: {name} must be ({L},) or ({B}, {L}), got {tuple(pos.shape)}")


def _rows(x):
    """x with a contiguous last dimension (x itself where it has one)."""
    return x if x.stride(3) == 1 or x.shape[3] == 1 else x.contiguous()


_POS = {torch.int32: _lib.POS_I32, torch.int64: _lib.POS_I64}
_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _like(x):
    """A new contiguous tensor of x's shape."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _heads(x, y, w, pos, g=None, gw=None):
    """The packed HclsmHeads of one tensor."""
    B, L, H, _ = x.shape
    sb, sl, sh, _ = x.stride()
    gb, gl, gh, _ = (0, 0, 0, 0) if g is None else g.stride()
    pb = pl = pd = pp = 0
    if pos is not None:
        pb, pl = (0, pos.stride(0)) if pos.dim() == 1 else pos.stride()
        pd, pp = _POS[pos.dtype], pos.data_ptr()
    return _lib.pack_heads(x.data_ptr(), 0 if g is None else g.data_ptr(), y.data_ptr(), 0 if w is None else w.data_ptr(),
                           0 if gw is None else gw.data_ptr(), pp, sb, sl, sh, gb, gl, gh, pb, pl, B, L, H,
                           0 if w is None else _CODE[w.dtype], pd)


def _plan_args(plan, back=False):
    """rot, layout, device pointer of the turns, amplitude."""
    if plan is None:
        return 0, _lib.ROTARY_HALF, None, 1.0
    return plan.rot_dim, plan._code, plan._turns.data_ptr() + (plan.rot_dim // 2 * 8 if back else 0), plan.amplitude


def _forward(tensors, plan, eps, norm, back=False):
    """tensors: [(x, w, positions)], one or two; returns the outputs."""
    ys, hs = [], []
    for x, w, pos in tensors:
        x = _rows(x)
        y = _like(x)
        ys.append(y)
        hs.append((_heads(x, y, w, pos), x))        # x: a copy has to live until the launch
    rot, layout, turns, amp = _plan_args(plan, back)
    x = hs[0][1]
    with on_device(x.device):
        rc = _lib.lib().hclsm_norm_rotary_forward(hs[0][0], hs[1][0] if len(hs) > 1 else None, x.shape[3], rot, layout,
                                                  turns, amp, eps, norm, _CODE[x.dtype], _lib.stream_of(x))
    if rc:
        _lib.check(rc, "hclsm_norm_rotary_forward")
    return ys


def _norm_backward(tensors, plan, eps):
    """tensors: [(x, w, positions, g, want gradient of w)], one or two; returns [(gx, gw or None)]."""
    out, hs = [], []
    for x, w, pos, g, want in tensors:
        x = _rows(x)
        g = _rows(g if g.dtype is x.dtype else g.to(x.dtype))
        gx, gw = _like(x), torch.empty_like(w) if want and w is not None else None
        out.append((gx, gw))
        hs.append((_heads(x, gx, w, pos, g, gw), x, g))
    rot, layout, turns, amp = _plan_args(plan)
    x = hs[0][1]
    L = _lib.lib()
    wsb = L.hclsm_norm_rotary_backward_workspace(x.shape[3], len(hs))
    ws = torch.empty(wsb, dtype=torch.uint8, device=x.device)
    with on_device(x.device):
        rc = L.hclsm_norm_rotary_backward(hs[0][0], hs[1][0] if len(hs) > 1 else None, x.shape[3], rot, layout, turns,
                                          amp, eps, _CODE[x.dtype], ws.data_ptr(), wsb, _lib.stream_of(x))
    if rc:
        _lib.check(rc, "hclsm_norm_rotary_backward")
    return out


class _Rotary(torch.autograd.Function):
    """The gradient of a rotation is the rotation back."""

    @staticmethod
    def forward(ctx, x, plan, positions):
        ctx.save_for_backward(positions)
        ctx.plan = plan
        ctx.dtype = x.dtype
        return _forward([(x, None, positions)], plan, 0.0, 0)[0]

    @staticmethod
    def backward(ctx, g):
        return once(_Rotary._back, ctx, g)

    @staticmethod
    def _back(ctx, g):
        (positions,) = ctx.saved_tensors
        if g.dtype is not ctx.dtype:
            g = g.to(ctx.dtype)
        return _forward([(g, None, positions)], ctx.plan, 0.0, 0, back=True)[0], None, None


def rotary_embedding(x: torch.Tensor, plan: RotaryPlan, positions: torch.Tensor | None = None) -> torch.Tensor:
    """x (B, L, H, dh) with the first plan.rot_dim elements of every head turned by its token's position."""
    require_gpu("rotary_embedding", x, positions, plan._turns if isinstance(plan, RotaryPlan) else None)
    _check_heads("rotary_embedding", "x", x)
    if plan is None:
        raise TypeError("rotary_embedding: plan must be a RotaryPlan, got NoneType")
    _check_plan("rotary_embedding", plan, x.shape[3])
    _check_positions("rotary_embedding", "positions", positions, x)
    if _no_node((x,)):
        return _forward([(x, None, positions)], plan, 0.0, 0)[0]
    return _Rotary.apply(x, plan, positions)


class _QKNormRotary(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, plan, positions, key_positions, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, key_positions)
        ctx.plan, ctx.eps = plan, eps
        ts = [(q, q_weight, positions)] + ([(k, k_weight, key_positions)] if k is not None else [])
        ys = _forward(ts, plan, eps, 1)
        return (ys[0], ys[1] if k is not None else None)

    @staticmethod
    def backward(ctx, gq, gk):
        return once(_QKNormRotary._back, ctx, gq, gk)

    @staticmethod
    def _back(ctx, gq, gk):
        q, k, wq, wk, pos, kpos = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads = [None] * 8
        ts, where = [], []
        for i, (x, w, p, g) in enumerate(((q, wq, pos, gq), (k, wk, kpos, gk))):
            if x is not None and (need[i] or need[2 + i]):
                ts.append((x, w, p, g, need[2 + i]))
                where.append(i)
        if ts:
            for i, (gx, gw) in zip(where, _norm_backward(ts, ctx.plan, ctx.eps)):
                grads[i], grads[2 + i] = gx, gw
        return tuple(grads)


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor | None, q_weight: torch.Tensor | None = None,
                   k_weight: torch.Tensor | None = None, plan: RotaryPlan | None = None,
                   positions: torch.Tensor | None = None, key_positions: torch.Tensor | None = None, *,
                   eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Root-mean-square norm of every head of q (B, L, H, dh) and k (B', L', H', dh), times q_weight / k_weight (dh,)
    (None: ones), then the plan's rotation (None: no rotation) by positions / key_positions.  k None: queries only
    (a step whose keys were prepared before).  Returns (q, k)."""
    fn = "qk_norm_rotary"
    require_gpu(fn, q, k, q_weight, k_weight, positions, key_positions,
                plan._turns if isinstance(plan, RotaryPlan) else None)
    _check_heads(fn, "q", q)
    _check_plan(fn, plan, q.shape[3])
    _check_positions(fn, "positions", positions, q)
    if k is not None:
        _check_heads(fn, "k", k)
        if k.dtype != q.dtype or k.shape[3] != q.shape[3]:
            raise ValueError(f"{fn}: q and k must share dtype and head size, got {q.dtype} {q.shape[3]} and {k.dtype} "
                             f"{k.shape[3]}")
        _check_positions(fn, "key_positions", key_positions, k)
    elif k_weight is not None or key_positions is not None:
        raise ValueError(f"{fn}: k_weight and key_positions need k")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        _check_weight(fn, name, w, q)
    if not eps >= 0:
        raise ValueError(f"{fn}: eps must be >= 0, got {eps}")
    if _no_node([t for t in (q, k, q_weight, k_weight) if t is not None]):
        ts = [(q, q_weight, positions)] + ([(k, k_weight, key_positions)] if k is not None else [])
        ys = _forward(ts, plan, float(eps), 1)
        return ys[0], (ys[1] if k is not None else None)
    return _QKNormRotary.apply(q, k, q_weight, k_weight, plan, positions, key_positions, float(eps))
