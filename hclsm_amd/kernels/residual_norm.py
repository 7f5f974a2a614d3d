"""Root-mean-square norm with the residual's addition (libhclsm_amd.so: hclsm_residual_norm_*).

    y, h = residual_rms_norm(x, residual, weight)                  # h = x + residual, y = norm(h) weight
    y8, scale, h = residual_rms_norm_fp8(x, residual, weight)      # y = y8 scale, for a product in 8 bits

The step between two layers of a residual stream in one pass: what the layer gave is added to the stream, and the next
layer's input is the norm of the sum.  The norm is that of h as it is returned (rounded to the stream's type), as it is
where a program adds first and normalises then.
"""

from __future__ import annotations

import torch

from hclsm_amd import _lib
from hclsm_amd.kernels._common import call_on, once, refuse_transforms, require_gpu
from hclsm_amd.kernels.ssm_scan_kernel import _no_node

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
MAX_COLUMNS = 16384
GROUPS = (32, 64, 128)
_INF = float("inf")
_BWD_BLOCKS = 1024          # most partial sums of the weight's gradient (hclsm_residual_norm_backward_workspace)


def _check(fn, x, residual, weight, eps):
    """One test of everything, and what is wrong if it fails."""
    shape, dt = x.shape, x.dtype
    if not (shape and dt in _CODE and 1 <= shape[-1] <= MAX_COLUMNS
            and (residual is None or (residual.shape == shape and residual.dtype in (dt, torch.float32)))
            and (weight is None or (weight.shape == shape[-1:] and weight.dtype in _CODE)) and 0 <= eps < _INF):
        _explain(fn, x, residual, weight, eps)


def _explain(fn, x, residual, weight, eps):
    if x.dim() < 1:
        raise ValueError(f"{fn}: x must be (..., D), got a scalar")
    if x.dtype not in _FLOATS:
        raise TypeError(f"{fn}: x must be bfloat16, float16 or float32, got {x.dtype}")
    D = x.shape[-1]
    if not 1 <= D <= MAX_COLUMNS:
        raise ValueError(f"{fn}: rows of 1 to {MAX_COLUMNS} elements, got {D}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"{fn}: residual must be {tuple(x.shape)}, got {tuple(residual.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{fn}: residual must be {x.dtype} or float32, got {residual.dtype}")
    if weight is not None and (tuple(weight.shape) != (D,) or weight.dtype not in _FLOATS):
        raise ValueError(f"{fn}: weight must be a float tensor of {D} elements, got {weight.dtype} {tuple(weight.shape)}")
    raise ValueError(f"{fn}: eps must be >= 0 and finite, got {eps}")


def _check_group(fn, x, group):
    if group is not None and (group not in GROUPS or x.shape[-1] % group):
        raise ValueError(f"{fn}: group must be None or one of {GROUPS} that divides {x.shape[-1]}, got {group}")


def _rows2d(t, D):
    """(rows, D) of a tensor, and the rows' stride: a view where the columns are contiguous and the rows evenly apart."""
    if t.is_contiguous():
        return t, D
    if t.dim() == 2 and (t.stride(1) == 1 or D == 1):
        return t, t.stride(0)
    return t.contiguous(), D


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _like(t, dtype=None):
    """A new contiguous tensor of t's shape."""
    return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


def _run(name, t, *args):
    """The library's entry on t's device and stream (its last argument)."""
    index = t.get_device()
    rc = call_on(index, getattr(_lib.lib(), name), *args, _lib.stream_of_device(index))
    if rc:
        _lib.check(rc, name)


def _forward(x, residual, weight, eps):
    D, code = x.shape[-1], _CODE[x.dtype]
    y, n = _like(x), x.numel() // D
    x, xs = _rows2d(x, D)
    if residual is None:
        h, r, rs, hc = None, None, 0, code
    else:
        h, hc = _like(residual), _CODE[residual.dtype]
        r, rs = _rows2d(residual, D)
    a = _lib.pack_residual(x.data_ptr(), _ptr(r), _ptr(weight), 0, 0, 0, y.data_ptr(), _ptr(h), 0, 0, 0, 0, xs, rs, 0, 0, 0,
                           n, D, 0, eps, code, hc, 0 if weight is None else _CODE[weight.dtype])
    _run("hclsm_residual_norm_forward", x, a)
    return y, h


def _forward_fp8(x, residual, weight, eps, group):
    D, code = x.shape[-1], _CODE[x.dtype]
    y, n = _like(x, torch.float8_e4m3fn), x.numel() // D
    scale = torch.empty((*x.shape[:-1], D // group if group else 1), dtype=torch.float32, device=x.device)
    x, xs = _rows2d(x, D)
    if residual is None:
        h, r, rs, hc = None, None, 0, code
    else:
        h, hc = _like(residual), _CODE[residual.dtype]
        r, rs = _rows2d(residual, D)
    if group:       # a group's lanes read whole vectors
        x, xs = _on_boundaries(x, xs)
        if r is not None:
            r, rs = _on_boundaries(r, rs)
    a = _lib.pack_residual(x.data_ptr(), _ptr(r), _ptr(weight), 0, 0, 0, y.data_ptr(), _ptr(h), scale.data_ptr(), 0, 0, 0, xs,
                           rs, 0, 0, 0, n, D, group, eps, code, hc, 0 if weight is None else _CODE[weight.dtype])
    _run("hclsm_residual_norm_fp8", x, a)
    return y, scale, h


def _on_boundaries(t, stride):
    if t.data_ptr() % 16 == 0 and stride * t.element_size() % 16 == 0:
        return t, stride
    return t.clone(memory_format=torch.contiguous_format), t.shape[-1]


def _backward(h, weight, gy, gh, eps, x_dtype, want_x, want_r, want_w):
    """Gradients of x, of the residual (None where it is that of x) and of the weight."""
    h_dtype, D = h.dtype, h.shape[-1]
    if gy is not None and gy.dtype is not x_dtype:
        gy = gy.to(x_dtype)
    if gh is not None and gh.dtype is not h_dtype:
        gh = gh.to(h_dtype)
    same = h_dtype is x_dtype
    n = h.numel() // D
    dx = _like(h, x_dtype) if want_x or (same and want_r) else None
    dr = _like(h) if want_r and not same else None
    dw = ws = None
    wsb = 0
    if want_w:
        dw = torch.empty_like(weight)
        wsb = (n if n < _BWD_BLOCKS else _BWD_BLOCKS) * D * 4
        ws = torch.empty(wsb + 16, dtype=torch.uint8, device=h.device)
    h, hs = _rows2d(h, D)
    gy, gys = (None, 0) if gy is None else _rows2d(gy, D)
    gh, ghs = (None, 0) if gh is None else _rows2d(gh, D)
    a = _lib.pack_residual(0, 0, _ptr(weight), h.data_ptr(), _ptr(gy), _ptr(gh), 0, 0, 0, _ptr(dx), _ptr(dr), _ptr(dw), 0, 0, hs,
                           gys, ghs, n, D, 0, eps, _CODE[x_dtype], _CODE[h_dtype], 0 if weight is None else _CODE[weight.dtype])
    _run("hclsm_residual_norm_backward", h, a, _ptr(ws), wsb)
    return dx, (dx if same else dr) if want_r else None, dw


class _ResidualNorm(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h = _forward(x, residual, weight, eps)
        if h is None:
            h = x           # an output too (a view of x): its gradient is added in the backward's one rounding
        ctx.save_for_backward(h, weight)
        ctx.eps, ctx.x_dtype = eps, x.dtype
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    def backward(ctx, gy, gh):
        return once(_ResidualNorm._back, ctx, gy, gh)

    @staticmethod
    def _back(ctx, gy, gh):
        if gy is None and gh is None:
            return None, None, None, None
        h, weight = ctx.saved_tensors
        x, r, w, _ = ctx.needs_input_grad
        dx, dr, dw = _backward(h, weight, gy, gh, ctx.eps, ctx.x_dtype, x, r, w)
        return dx if x else None, dr, dw, None


def residual_rms_norm(x: torch.Tensor, residual: torch.Tensor | None = None, weight: torch.Tensor | None = None, *,
                      eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = x + residual and y = h / sqrt(mean(h^2) + eps) * weight over the last dimension.

    x (..., D), bfloat16, float16 or float32, 1 <= D <= 16384; residual: x's shape, x's type or float32, or None (then h is
    x, or a view of it where gradients are recorded); weight (D,) of any of the float types, None: ones.  Rows of (rows, D) views may lie any distance apart; other
    views are copied.  y has x's type, h the residual's.  Differentiable in all three, through both outputs; float32 between
    the loads and the one rounding of each output (a row whose squares add up to more than float32 holds, 3.4e38, gives
    zeros)."""
    fn = "residual_rms_norm"
    require_gpu(fn, x, residual, weight)
    eps = float(eps)
    _check(fn, x, residual, weight, eps)
    if weight is not None:
        weight = weight.contiguous()
    if _no_node([t for t in (x, residual, weight) if t is not None]):
        y, h = _forward(x, residual, weight, eps)
    else:
        return _ResidualNorm.apply(x, residual, weight, eps)
    return y, (x if h is None else h)


def residual_rms_norm_fp8(x: torch.Tensor, residual: torch.Tensor | None = None, weight: torch.Tensor | None = None, *,
                          eps: float = 1e-6, group: int | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y8, scale, h): ``residual_rms_norm`` with y as y8 * scale, y8 of torch.float8_e4m3fn.

    group None: one scale for a row, scale (..., 1); 32, 64 or 128: one for each so many columns, scale (..., D / group).
    scale = max(max |y|, 2^-100) / 448, y8 = y / scale rounded to the nearest value.  A NaN makes its row NaN, and so does
    an infinity with one scale for a row; with groups, it makes its own group NaN and the row's other groups zeros (as
    ``residual_rms_norm`` has them: the root is infinite).  For inference: tensors that require grad are refused while gradients are recorded, and so are tangents,
    function transforms and traces (torch.ops.hclsm_hip.residual_rms_norm_fp8 can be traced)."""
    fn = "residual_rms_norm_fp8"
    require_gpu(fn, x, residual, weight)
    refuse_transforms(fn, x, residual, weight)
    eps = float(eps)
    _check(fn, x, residual, weight, eps)
    _check_group(fn, x, group)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight)):
        raise RuntimeError(f"{fn}: 8-bit outputs have no gradient; use residual_rms_norm, or torch.no_grad()")
    y, scale, h = _forward_fp8(x, residual, None if weight is None else weight.contiguous(), eps, group or 0)
    return y, scale, (x if h is None else h)
