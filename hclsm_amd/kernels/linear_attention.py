"""Linear attention with a decay for each head (libhclsm_amd.so: hclsm_linear_attention_*).

    out, state = linear_attention(q, k, v, log_decay, return_state=True)      # a prompt, or a training step
    out = linear_attention_step(q, k, v, log_decay, state)                    # one token, the state updated in place

S_t = exp(log_decay) S_{t-1} + k_t v_t^T and out_t = scale q_t^T S_t, with one float32 state of dk x dv for each head.  A
time mixer like the selective scan (``ssm_scan_fn``; the reference's kernels/ssm_scan_kernel.py) with a state of matrices
and products between the tokens of a chunk, for the tracks of a clip or the tokens of a long stream.
"""

from __future__ import annotations

import torch

from hclsm_amd import _lib
from hclsm_amd.kernels._common import call_on, once, refuse_transforms, require_gpu
from hclsm_amd.kernels.ssm_scan_kernel import _no_node

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
MAX_HEAD_DIM = 256
_MAX_HEADS = 1 << 20        # heads of a call, B H
_MAX_ROW = 1 << 23          # elements of a token, H max(dk, dv)
_FAR = 1 << 23              # elements between tokens


def _check(fn, q, k, v, log_decay, scale, token):
    """q (B, [L,] H, dk), k and v (B, [L,] Hk, dk / dv); token: no L.  One test of everything, and what is wrong if it fails."""
    qs, ks, vs, dt = q.shape, k.shape, v.shape, q.dtype
    n = len(qs)
    if not (n == (3 if token else 4) and len(ks) == n and len(vs) == n and dt in _CODE and k.dtype is dt and v.dtype is dt
            and ks[:-2] == qs[:-2] and ks[-1] == qs[-1] and vs[:-1] == ks[:-1] and 1 <= ks[-2] <= qs[-2] and qs[-2] % ks[-2] == 0
            and 8 <= qs[-1] <= MAX_HEAD_DIM and qs[-1] % 8 == 0 and 8 <= vs[-1] <= MAX_HEAD_DIM and vs[-1] % 8 == 0
            and qs[0] * qs[-2] <= _MAX_HEADS and qs[-2] * max(qs[-1], vs[-1]) < _MAX_ROW
            and log_decay.shape == qs[-2:-1] and log_decay.dtype is torch.float32 and 1e-38 <= scale <= 3e38):
        _explain(fn, q, k, v, log_decay, scale, token)
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{fn}: log_decay has no gradient here; pass log_decay.detach()")


def _explain(fn, q, k, v, log_decay, scale, token):
    dims, shape = (3, "(B, H, d)") if token else (4, "(B, L, H, d)")
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != dims:
            raise ValueError(f"{fn}: {name} must be {shape}, got shape {tuple(t.shape)}")
        if t.dtype not in _FLOATS or t.dtype != q.dtype:
            raise TypeError(f"{fn}: q, k, v must share one dtype among bfloat16, float16, float32, got {name} {t.dtype}")
    H, dk, Hk, dv = q.shape[-2], q.shape[-1], k.shape[-2], v.shape[-1]
    if k.shape[:-2] != q.shape[:-2] or k.shape[-1] != dk or v.shape[:-1] != k.shape[:-1]:
        raise ValueError(f"{fn}: k must be {(*q.shape[:-2], 'Hk', dk)} and v {(*q.shape[:-2], 'Hk', 'dv')}, got "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    if Hk < 1 or H < 1 or H % Hk:
        raise ValueError(f"{fn}: {H} heads cannot share {Hk} key heads")
    for name, d in (("dk", dk), ("dv", dv)):
        if not 8 <= d <= MAX_HEAD_DIM or d % 8:
            raise ValueError(f"{fn}: heads of 8, 16, .. {MAX_HEAD_DIM} elements, got {name} = {d}")
    if q.shape[0] * H > _MAX_HEADS:
        raise ValueError(f"{fn}: at most {_MAX_HEADS} heads in a call, got {q.shape[0]} x {H}")
    if H * max(dk, dv) >= _MAX_ROW:
        raise ValueError(f"{fn}: fewer than {_MAX_ROW} elements in a token, got {H} x {max(dk, dv)}")
    if tuple(log_decay.shape) != (H,) or log_decay.dtype != torch.float32:
        raise ValueError(f"{fn}: log_decay must be ({H},) float32, got {tuple(log_decay.shape)} {log_decay.dtype}")
    raise ValueError(f"{fn}: scale must be positive, as a float32 too, got {scale}")


def _check_index(fn, name, t, B):
    if t is None:
        return
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{fn}: {name} must be int32 or int64, got {t.dtype}")
    if tuple(t.shape) != (B,):
        raise ValueError(f"{fn}: {name} must be ({B},), got {tuple(t.shape)}")


def _check_first(fn, state, q, v):
    """A state (or its gradient) in front of or behind a sequence."""
    want = (q.shape[0], q.shape[2], q.shape[3], v.shape[3])
    if state is not None and (state.shape != want or state.dtype is not torch.float32):
        raise ValueError(f"{fn}: initial_state must be {want} float32, got {tuple(state.shape)} {state.dtype}")


def _index(t):
    return t if t is None or t.stride(0) == 1 or t.shape[0] < 2 else t.contiguous()


def _index_code(t):
    return _lib.POS_I64 if t is not None and t.dtype is torch.int64 else _lib.POS_I32


def _rows(t):
    """t with rows on 16-byte boundaries and near enough to each other (t itself where they are): the kernels' offsets from
    a chunk's first row are 31 bits."""
    n = 16 // t.element_size()
    if t.is_contiguous() and t.data_ptr() % 16 == 0:        # (heads are multiples of 8 elements, tokens smaller than _FAR)
        return t
    sb, sl, sh, s = t.stride()
    B, L, H, _ = t.shape
    if (s == 1 and t.data_ptr() % 16 == 0 and (sb % n == 0 or B == 1) and (L == 1 or (sl % n == 0 and sl < _FAR))
            and (sh % n == 0 or H == 1)):
        return t
    if not t.is_contiguous():
        return t.contiguous()
    return t.clone(memory_format=torch.contiguous_format) if t.data_ptr() % 16 else t


def _strides(t):
    sb, sl, sh, _ = t.stride()
    B, L, H, _ = t.shape
    return sb if B > 1 else 0, sl if L > 1 else 0, sh if H > 1 else 0


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _run(name, t, *args):
    """The library's entry on t's device and stream (its last argument)."""
    index = t.get_device()
    rc = call_on(index, getattr(_lib.lib(), name), *args, _lib.stream_of_device(index))
    if rc:
        _lib.check(rc, name)


_WORKSPACE: dict = {}       # sizes -> bytes (a function of the sizes alone)


def _workspace(q, k, v, backward):
    key = (*q.shape, k.shape[2], v.shape[3], q.dtype, backward)
    n = _WORKSPACE.get(key)
    if n is None:
        B, L, H, dk = q.shape
        n = int(_lib.lib().hclsm_linear_attention_workspace(B, L, H, k.shape[2], dk, v.shape[3], _CODE[q.dtype], backward))
        if n < 0:
            _lib.check(n, "hclsm_linear_attention_workspace")
        if len(_WORKSPACE) > 4096:
            _WORKSPACE.clear()
        _WORKSPACE[key] = n
    return (torch.empty(n, dtype=torch.uint8, device=q.device) if n else None), n


def _forward(q, k, v, log_decay, s0, lens, scale, want_state):
    q, k, v = _rows(q), _rows(k), _rows(v)
    B, L, H, dk = q.shape
    dv = v.shape[3]
    out = torch.empty((B, L, H, dv), dtype=q.dtype, device=q.device)
    s1 = torch.empty((B, H, dk, dv), dtype=torch.float32, device=q.device) if want_state else None
    ws, n = _workspace(q, k, v, 0)
    x = _lib.pack_linear(q.data_ptr(), k.data_ptr(), v.data_ptr(), 0, log_decay.data_ptr(), _ptr(s0), _ptr(s1), 0, 0,
                         out.data_ptr(), 0, 0, 0, _ptr(lens), *_strides(q), *_strides(k), *_strides(v), 0, 0, 0, B, L, H,
                         k.shape[2], dk, dv, scale, _CODE[q.dtype], _index_code(lens))
    _run("hclsm_linear_attention_forward", q, x, _ptr(ws), n)
    return out, s1


def _backward(q, k, v, log_decay, s0, lens, scale, g, gs, want):
    """Gradients of q, k, v and the first state, None where not in `want`.  g, gs: gradients of the outputs, None: zero."""
    B, L, H, dk = q.shape
    dv = v.shape[3]
    if g is None:
        g = torch.zeros((B, L, H, dv), dtype=q.dtype, device=q.device)
    elif g.dtype is not q.dtype:
        g = g.to(q.dtype)
    q, k, v, g = _rows(q), _rows(k), _rows(v), _rows(g)
    gs = None if gs is None else gs.contiguous()
    new = lambda t, w: torch.empty(t.shape, dtype=t.dtype, device=t.device) if w else None
    dq, dk_, dv_ = new(q, want[0]), new(k, want[1]), new(v, want[2])
    ds = torch.empty((B, H, dk, dv), dtype=torch.float32, device=q.device) if want[3] else None
    ws, n = _workspace(q, k, v, 1)
    x = _lib.pack_linear(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), log_decay.data_ptr(), _ptr(s0), 0, _ptr(gs),
                         _ptr(ds), 0, _ptr(dq), _ptr(dk_), _ptr(dv_), _ptr(lens), *_strides(q), *_strides(k), *_strides(v),
                         *_strides(g), B, L, H, k.shape[2], dk, dv, scale, _CODE[q.dtype], _index_code(lens))
    _run("hclsm_linear_attention_backward", q, x, _ptr(ws), n)
    return dq, dk_, dv_, ds


class _LinearAttention(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, s0, log_decay, lens, scale, want_state):
        out, s1 = _forward(q, k, v, log_decay, s0, lens, scale, want_state)
        ctx.save_for_backward(q, k, v, s0, log_decay, lens)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, s1

    @staticmethod
    def backward(ctx, g, gs):
        return once(_LinearAttention._back, ctx, g, gs)

    @staticmethod
    def _back(ctx, g, gs):
        q, k, v, s0, log_decay, lens = ctx.saved_tensors
        if g is None and gs is None:
            return (None,) * 8
        return (*_backward(q, k, v, log_decay, s0, lens, ctx.scale, g, gs, ctx.needs_input_grad[:4]), None, None, None, None)


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *,
                     initial_state: torch.Tensor | None = None, seq_lens: torch.Tensor | None = None,
                     scale: float | None = None, return_state: bool = False):
    """out_t = scale q_t^T S_t with S_t = exp(log_decay) S_{t-1} + k_t v_t^T, for every head.

    q (B, L, H, dk); k (B, L, Hk, dk) and v (B, L, Hk, dv): head h reads key head h // (H // Hk).  One dtype among bfloat16,
        float16, float32; dk and dv multiples of 8 up to 256; any strides (rows that are not contiguous or not on 16-byte
        boundaries, or very far apart, are copied).  B H is at most 2^20, H max(dk, dv) below 2^23.
    log_decay (H,) float32, at most 0 (0 sums without decay, -inf keeps the token itself alone); a constant: it has no
        gradient here, and one that requires grad is refused.
    initial_state (B, H, dk, dv) float32: the state in front of the first token; None: zeros.
    seq_lens (B,) int32 or int64: tokens from seq_lens[b] on are not read (they may hold anything), give zeros, take part
        in no gradient and leave the state as it is.  Live tokens are to be finite: outputs of up to 63 tokens before one
        that is not may be NaN too (tokens are taken in chunks).
    scale: dk ** -0.5 if None; positive.

    Returns out (B, L, H, dv), and with return_state the state behind each row's last live token, (B, H, dk, dv) float32,
    for ``linear_attention_step`` or the next call.  Differentiable in q, k, v and initial_state, through both outputs; the
    same inputs give the same bits.  States and sums are float32; what is rounded in between for the matrix products keeps 16 bits
    (24 for float32 inputs and for the state)."""
    fn = "linear_attention"
    require_gpu(fn, q, k, v, log_decay, initial_state, seq_lens)
    if scale is None:
        scale = q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0
    scale = float(scale)
    _check(fn, q, k, v, log_decay, scale, False)
    _check_index(fn, "seq_lens", seq_lens, q.shape[0])
    _check_first(fn, initial_state, q, v)
    log_decay, lens = log_decay.contiguous(), _index(seq_lens)
    s0 = None if initial_state is None else initial_state.contiguous()
    if _no_node((q, k, v) if s0 is None else (q, k, v, s0)):
        out, s1 = _forward(q, k, v, log_decay, s0, lens, scale, return_state)
    else:
        out, s1 = _LinearAttention.apply(q, k, v, s0, log_decay, lens, scale, return_state)
    return (out, s1) if return_state else out


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor, *,
                          rows: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """One token of each of B streams: state = exp(log_decay) state + k v^T in place, out = scale q^T state.

    q (B, H, dk); k (B, Hk, dk) and v (B, Hk, dv), as ``linear_attention``'s without L, of any strides.
    state (N, H, dk, dv) float32, the heads of one state contiguous, on 16-byte boundaries: updated in place.
        A graph that has saved it (linear_attention's initial_state) raises in its backward, as behind torch's own writes.
    rows (B,) int32 or int64: which state is each stream's; None: stream b has state b, and N is B.  A row that is negative or
        not below N pads the batch: it gives zeros and touches no state.  Rows must differ from each other (of a state
        that two streams name, neither's update is certain).
    Returns out (B, H, dv).  For inference: tensors that require grad are refused while gradients are recorded, and so are
    tangents, function transforms and traces (torch.ops.hclsm_hip.linear_attention_step can be traced)."""
    fn = "linear_attention_step"
    require_gpu(fn, q, k, v, log_decay, state, rows)
    refuse_transforms(fn, q, k, v, log_decay, state)
    if scale is None:
        scale = q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0
    scale = float(scale)
    _check(fn, q, k, v, log_decay, scale, True)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad):
        raise RuntimeError(f"{fn}: the step has no gradient (it updates the state in place); use linear_attention, or "
                           "torch.no_grad()")
    B, H, dk = q.shape
    if rows is not None:
        _check_index(fn, "rows", rows, B)
    _check_state(fn, state, B if rows is None else None, H, dk, v.shape[2])
    torch.autograd.graph.increment_version(state)
    return _step(q, k, v, log_decay.contiguous(), state, _index(rows), scale)


def _check_state(fn, state, N, H, dk, dv):
    shape = state.shape
    if (len(shape) != 4 or shape[1] != H or shape[2] != dk or shape[3] != dv or state.dtype is not torch.float32
            or (N is not None and shape[0] != N)):
        raise ValueError(f"{fn}: state must be ({'N' if N is None else N}, {H}, {dk}, {dv}) float32, got "
                         f"{tuple(shape)} {state.dtype}")
    sb, sh, sr, sc = state.stride()
    if (sc != 1 or sr != dv or (sh != dk * dv and H > 1) or state.data_ptr() % 16
            or (shape[0] > 1 and (sb % 4 or sb < H * dk * dv))) and state.numel():
        raise ValueError(f"{fn}: the heads of a state must be contiguous, on 16-byte boundaries, and states apart (it is "
                         f"updated in place), got strides {state.stride()}")


def _step(q, k, v, log_decay, state, rows, scale):
    qb, qh, qe = q.stride()
    kb, kh, ke = k.stride()
    vb, vh, ve = v.stride()
    if qe != 1 or ke != 1 or ve != 1:
        return _step(q.contiguous(), k.contiguous(), v.contiguous(), log_decay, state, rows, scale)
    B, H, dk = q.shape
    _, Hk, dv = v.shape
    out = q.new_empty((B, H, dv))
    x = _lib.pack_step(q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), state.data_ptr(), _ptr(rows),
                       out.data_ptr(), qb, qh, kb, kh, vb, vh, state.stride(0) if state.shape[0] > 1 else 0, state.shape[0], B, H,
                       Hk, dk, dv, scale, _CODE[q.dtype], _index_code(rows))
    _run("hclsm_linear_attention_step", q, x)
    return out
