"""Argument checks shared by the hclsm_amd kernel wrappers."""

from __future__ import annotations

import contextlib

import torch


def require_gpu(fn_name: str, *tensors: "torch.Tensor | None") -> torch.device:
    """All tensors must live on one ROCm GPU; there is no CPU path."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(
                f"hclsm_amd.{fn_name}: tensors must be on a ROCm GPU (got a {t.device} tensor). "
                "hclsm_amd has no CPU implementation; move the inputs to 'cuda'.")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"hclsm_amd.{fn_name}: tensors are on different devices ({dev} and {t.device})")
    if dev is None:
        raise RuntimeError(f"hclsm_amd.{fn_name}: no tensor arguments")
    return dev


def common_float_dtype(*tensors: torch.Tensor) -> torch.dtype:
    """The kernels' I/O element type: shared dtype if all agree, else float32."""
    dts = {t.dtype for t in tensors if t is not None}
    if len(dts) == 1:
        (dt,) = dts
        if dt in (torch.float32, torch.bfloat16, torch.float16):
            return dt
    return torch.float32


def once(back, ctx, *grads):
    """back(ctx, *grads), which cannot be differentiated again: where a graph of the gradients is asked for (create_graph),
    differentiating it raises, and a gradient with a tangent is refused.  Elsewhere without the wrapper, which costs several us."""
    if torch.autograd.forward_ad._current_level >= 0:
        for g in grads:
            if g is not None and torch.autograd.forward_ad.unpack_dual(g).tangent is not None:
                raise RuntimeError("hclsm_amd: a gradient has a tangent, and there is no forward-mode derivative of this backward")
    if not torch.is_grad_enabled():
        return back(ctx, *grads)
    from torch.autograd.function import once_differentiable
    return once_differentiable(back)(ctx, *grads)


def refuse_transforms(fn_name: str, *tensors: "torch.Tensor | None") -> None:
    """For a call without an autograd function: refuse what does not see what the library does and would lose it without a
    word, tangents of forward-mode AD, function transforms and traces."""
    if torch.jit.is_tracing():
        raise RuntimeError(f"hclsm_amd.{fn_name}: a trace does not record this call; use torch.ops.hclsm_hip.{fn_name} in it")
    transforms, level = torch._C._are_functorch_transforms_active(), torch.autograd.forward_ad._current_level
    if not transforms and level < 0:
        return
    for t in tensors:
        if t is None:
            continue
        if transforms and torch._C._functorch.is_functorch_wrapped_tensor(t):
            raise RuntimeError(f"hclsm_amd.{fn_name}: no function transform (torch.func) goes through this call")
        if level >= 0 and torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"hclsm_amd.{fn_name}: an input has a tangent, and there is no forward-mode gradient here")


_SAME_DEVICE = contextlib.nullcontext()


def on_device(dev: torch.device):
    """Context in which a launch for tensors on ``dev`` is made: HIP launches go to the current device."""
    return _SAME_DEVICE if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def call_on(index: int, fn, *args):
    """fn(*args) with device ``index`` as the current one (``on_device`` without the cost of a context where it is)."""
    if torch.cuda.current_device() == index:
        return fn(*args)
    with torch.cuda.device(index):
        return fn(*args)


class HipFallbackWarning(UserWarning):
    """A call ran the reference's math as torch ops on the GPU instead of an hclsm_amd kernel (autograd through a
    forward-only kernel, or a module structure / shape the kernel does not take)."""


_WARNED: set = set()


def warn_fallback(fn_name: str, reason: str) -> None:
    """Warn (once per function and reason) that fn_name is running torch ops instead of its HIP kernel.  The
    pair is recorded only after the warning was issued, so under ``warnings.simplefilter("error",
    HipFallbackWarning)`` every such call raises."""
    import warnings
    key = (fn_name, reason)
    if key in _WARNED:
        return
    warnings.warn(f"hclsm_amd.{fn_name}: running the reference math as torch ops on the GPU: {reason}",
                  HipFallbackWarning, stacklevel=3)
    _WARNED.add(key)
