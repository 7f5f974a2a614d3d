"""Attention of queries against keys and values of another length (libhclsm_amd.so: hclsm_cross_attention_*).

    out = cross_attention(q, k, v)                       # q (B, Lq, H, dh), k and v (B, Lk, Hk, dh)

Slots or learned goal queries against the tokens of an encoder or the events of a clip: the attention core of
``nn.MultiheadAttention`` with keys of their own (the reference's dynamics/level2_goal.py:50,63 and
perception/multimodal_fuser.py:40; projections stay outside), with key heads shared by groups of query heads, lengths per
batch row, a key padding mask, gradients, and a form for few queries that splits the keys over the GPU.
"""

from __future__ import annotations

import warnings

import torch

from hclsm_amd import _lib
from hclsm_amd.kernels._common import on_device, once, require_gpu
from hclsm_amd.kernels.ssm_scan_kernel import _no_node

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
MAX_HEAD_DIM = 256


def _check(q, k, v, key_padding_mask, key_lens, query_lens, scale):
    fn = "cross_attention"
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"{fn}: {name} must be (B, L, H, dh), got shape {tuple(t.shape)}")
        if t.dtype not in _FLOATS or t.dtype != q.dtype:
            raise TypeError(f"{fn}: q, k, v must share one dtype among bfloat16, float16, float32, got {name} {t.dtype}")
    B, Lq, H, dh = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != dh:
        raise ValueError(f"{fn}: k and v must be ({B}, Lk, Hk, {dh}), got {tuple(k.shape)} and {tuple(v.shape)}")
    Lk, Hk = k.shape[1], k.shape[2]
    if Hk < 1 or H % Hk:
        raise ValueError(f"{fn}: {H} query heads cannot share {Hk} key heads")
    if not 8 <= dh <= MAX_HEAD_DIM or dh % 8:
        raise ValueError(f"{fn}: heads of 8, 16, .. {MAX_HEAD_DIM} elements, got {dh}")
    if key_padding_mask is not None and tuple(key_padding_mask.shape) != (B, Lk):
        raise ValueError(f"{fn}: key_padding_mask must be ({B}, {Lk}), got {tuple(key_padding_mask.shape)}")
    for name, t in (("key_lens", key_lens), ("query_lens", query_lens)):
        if t is None:
            continue
        if t.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{fn}: {name} must be int32 or int64, got {t.dtype}")
        if tuple(t.shape) != (B,):
            raise ValueError(f"{fn}: {name} must be ({B},), got {tuple(t.shape)}")
    if not 1e-45 <= scale <= 2e38:
        raise ValueError(f"{fn}: scale must be positive, as a float32 too, and at most 2e38, got {scale}")


def _masks(key_padding_mask, key_lens, query_lens):
    """The masks as the kernels read them: bytes with contiguous rows, contiguous lengths."""
    pad = key_padding_mask
    if pad is not None:
        if pad.is_floating_point():
            warnings.warn("cross_attention: a key_padding_mask of a float type is read as flags (nonzero = ignore that key), "
                          "not added to the scores as nn.MultiheadAttention would; pass mask != 0 if that is meant",
                          UserWarning, stacklevel=3)
        if pad.dtype not in (torch.bool, torch.uint8):
            pad = pad != 0
        if pad.stride(1) != 1:
            pad = pad.contiguous()
    return (pad, key_lens if key_lens is None or key_lens.stride(0) == 1 else key_lens.contiguous(),
            query_lens if query_lens is None or query_lens.stride(0) == 1 else query_lens.contiguous())


def _rows(t, keys=False):
    """t with rows on 16-byte boundaries and near enough to each other (t itself where they are).  The kernels' offsets from a
    tile's first row are 31 bits: of keys and values a tile has one head, of queries all heads that share a key head."""
    n = 16 // t.element_size()
    sb, sl, sh, s = t.stride()
    B, L, H, _ = t.shape
    if (s == 1 and t.data_ptr() % 16 == 0 and (sb % n == 0 or B == 1)
            and (L == 1 or (sl % n == 0 and (sl < 1 << 20 or (keys and sl < 1 << 22))))
            and (H == 1 or (sh % n == 0 and (keys or sh * H < 1 << 28)))):
        return t
    if not t.is_contiguous():
        return t.contiguous()
    return t.clone(memory_format=torch.contiguous_format) if t.data_ptr() % 16 else t


_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_WORKSPACE: dict = {}       # sizes -> bytes (a function of the sizes alone)


def _strides(t):
    sb, sl, sh, _ = t.stride()
    B, L, H, _ = t.shape
    return sb if B > 1 else 0, sl if L > 1 else 0, sh if H > 1 else 0


def _pack(q, k, v, out, out_lo, lse, masks, scale, g=None, dq=None, dk=None, dv=None):
    """The packed HclsmCrossAttention of a call."""
    pad, klens, qlens = masks
    B, Lq, H, dh = q.shape
    p = lambda t: 0 if t is None else t.data_ptr()
    code = lambda t: _lib.POS_I64 if t is not None and t.dtype is torch.int64 else _lib.POS_I32
    return _lib.pack_cross(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), p(g), out.data_ptr(), p(out_lo), p(lse), p(dq), p(dk), p(dv), p(pad),
        p(klens), p(qlens), *_strides(q), *_strides(k), *_strides(v), *((0, 0, 0) if g is None else _strides(g)),
        pad.stride(0) if pad is not None and B > 1 else 0, B, Lq, k.shape[1], H, k.shape[2], dh, scale, _CODE[q.dtype],
        code(klens), code(qlens))


def _workspace(q, k, backward):
    key = (*q.shape, k.shape[1], k.shape[2], q.dtype, backward)
    n = _WORKSPACE.get(key)
    if n is None:
        B, Lq, H, dh = q.shape
        n = int(_lib.lib().hclsm_cross_attention_workspace(B, Lq, k.shape[1], H, k.shape[2], dh, _CODE[q.dtype], backward))
        if n < 0:
            _lib.check(n, "hclsm_cross_attention_workspace")
        if len(_WORKSPACE) > 4096:
            _WORKSPACE.clear()
        _WORKSPACE[key] = n
    return (torch.empty(n, dtype=torch.uint8, device=q.device) if n else None), n


def _like(t):
    """A new contiguous tensor of t's shape."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _forward(q, k, v, masks, scale, want_lse, want_lo):
    q, k, v = _rows(q), _rows(k, True), _rows(v, True)
    B, Lq, H, _ = q.shape
    out = _like(q)
    lo = _like(q) if want_lo else None
    lse = torch.empty((B, H, Lq), dtype=torch.float32, device=q.device) if want_lse else None
    ws, n = _workspace(q, k, 0)
    x = _pack(q, k, v, out, lo, lse, masks, scale)
    with on_device(q.device):
        rc = _lib.lib().hclsm_cross_attention_forward(x, None if ws is None else ws.data_ptr(), n, _lib.stream_of(q))
    if rc:
        _lib.check(rc, "hclsm_cross_attention_forward")
    return out, lse, lo


def _backward(q, k, v, out, lo, lse, g, masks, scale, want_q=True, want_kv=True):
    q, k, v, g = _rows(q), _rows(k, True), _rows(v, True), _rows(g if g.dtype is q.dtype else g.to(q.dtype))
    dq, dk, dv = _like(q) if want_q else None, _like(k) if want_kv else None, _like(v) if want_kv else None
    ws, n = _workspace(q, k, 1)
    x = _pack(q, k, v, out, lo, lse, masks, scale, g, dq, dk, dv)
    with on_device(q.device):
        rc = _lib.lib().hclsm_cross_attention_backward(x, None if ws is None else ws.data_ptr(), n, _lib.stream_of(q))
    if rc:
        _lib.check(rc, "hclsm_cross_attention_backward")
    return dq, dk, dv


class _CrossAttention(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, masks, scale):
        # 16-bit outputs: what their rounding dropped is kept too, for the backward's sum(g out)
        out, lse, lo = _forward(q, k, v, masks, scale, True, q.dtype is not torch.float32)
        ctx.save_for_backward(q, k, v, out, lo, lse, *masks)
        ctx.scale = scale
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    def backward(ctx, g, _):
        return once(_CrossAttention._back, ctx, g)

    @staticmethod
    def _back(ctx, g):
        q, k, v, out, lo, lse, *masks = ctx.saved_tensors
        need = ctx.needs_input_grad
        dq, dk, dv = _backward(q, k, v, out, lo, lse, g, masks, ctx.scale, need[0], need[1] or need[2])
        return dq, dk if need[1] else None, dv if need[2] else None, None, None


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, key_padding_mask: torch.Tensor | None = None,
                    key_lens: torch.Tensor | None = None, query_lens: torch.Tensor | None = None,
                    scale: float | None = None, return_lse: bool = False):
    """softmax(scale q k^T) v for every head.

    q (B, Lq, H, dh); k, v (B, Lk, Hk, dh): head h reads key head h // (H // Hk).  One dtype among bfloat16, float16,
        float32; dh a multiple of 8 up to 256; any strides (rows that are not contiguous, not on 16-byte boundaries
        or very far apart are copied; a batch of stride 0 is read as it stands).
    key_padding_mask (B, Lk), True (or nonzero) = ignore that key, nn.MultiheadAttention's convention for boolean masks.  A
        mask of a float type is read the same way, with a warning: it is not added to the scores.  key_lens (B,) int32 or
        int64: keys from key_lens[b] on are ignored.  What ignored keys hold, NaN and infinities among it, has no effect.
    query_lens (B,): queries from query_lens[b] on give zeros, and take part in no gradient.
    scale: dh ** -0.5 if None; positive.

    Returns out (B, Lq, H, dh) [, lse (B, H, Lq) float32: the softmax's log-denominator, not differentiable].  A query
    with no key to read gives zeros (lse -inf) and zero gradients (slots_attention gives NaN there).  Differentiable in
    q, k and v; the same inputs give the same bits.  Scores, softmax and sums are float32; with 16-bit inputs the
    weights (and in the backward the scores' gradients) are rounded to the inputs' type for the matrix products, with what
    the rounding drops as a second operand where a key head has at most 16 query rows (32 of heads up to 64, and in the
    backward of heads up to 128) or there are at most 32 keys; float16 gradients of scores are rounded relative to the
    largest of their row or key, whatever their size."""
    require_gpu("cross_attention", q, k, v, key_padding_mask, key_lens, query_lens)
    if scale is None:
        scale = q.shape[-1] ** -0.5
    scale = float(scale)
    _check(q, k, v, key_padding_mask, key_lens, query_lens, scale)
    masks = _masks(key_padding_mask, key_lens, query_lens)
    if _no_node((q, k, v)):
        out, lse, _ = _forward(q, k, v, masks, scale, return_lse, False)
    else:
        out, lse = _CrossAttention.apply(q, k, v, masks, scale)
    return (out, lse) if return_lse else out
