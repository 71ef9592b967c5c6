"""Torch-side plumbing shared by the op wrappers: dtype codes, stream, checks."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad as _forward_ad

from .. import _lib

_DTYPE = {torch.float32: _lib.HXM_F32, torch.bfloat16: _lib.HXM_BF16, torch.float16: _lib.HXM_F16}


def dtype_code(t: torch.Tensor) -> int:
    try:
        return _DTYPE[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}") from None


def require_cuda(*tensors, who: str):
    """The kernels run only on a CUDA device; there is no CPU fallback."""
    first = index = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{who}: tensors must be on a CUDA device (got {t.device}); "
                               "this package has no CPU path")
        if first is None:
            first, index = t, t.get_device()
        elif t.get_device() != index:
            raise RuntimeError(f"{who}: tensors on different devices ({first.device} vs {t.device})")
    return None if first is None else first.device


# The raw cudaStream_t of a device's current stream: the Stream object around it costs 2 us a call.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)  # of tensors, so CUDA is initialised


def stream_of(device) -> int:
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


class _Here:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def on_device(device):
    """A context in which ``device`` is the current CUDA device (launches go to the current device's
    context, whatever stream they name); free when it already is."""
    return _HERE if device.index == _device() else torch.cuda.device(device)


def once_only(who):
    """Raises in a backward that is itself being differentiated (create_graph=True): its kernels record nothing."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{who}: its gradient cannot be differentiated again")


def no_tangents(who, *tensors):
    """Raises where a tensor carries a forward-mode tangent: the kernels would drop it without a word."""
    if _forward_ad._current_level < 0:  # outside of dual_level, torch.func.jvp and the like
        return
    for t in tensors:
        if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{who}: has no forward-mode derivative")


def ptr(t):
    return None if t is None else t.data_ptr()


def strides(t, n):
    return (0,) * n if t is None else tuple(t.stride())


def f32_param(t):
    """``t`` as a contiguous fp32 tensor, for small parameters (weights, biases) that the
    kernels read in fp32.  A bf16 parameter's fp32 copy is kept on the tensor and reused while
    the tensor is unchanged (same storage and version), so inference calls launch no cast
    kernel; with autograd recording for ``t`` the cast is a fresh differentiable op, and a copy
    first made during a CUDA-graph capture is not kept."""
    if t is None:
        return None
    if t.dtype == torch.float32 and t.is_contiguous():
        return t
    if torch.is_grad_enabled() and t.requires_grad:
        return t.float().contiguous()
    key = (t.data_ptr(), t._version, tuple(t.shape), t.stride())
    hit = getattr(t, "_hxm_f32", None)
    if hit is not None and hit[0] == key:
        return hit[1]
    v = t.detach().float().contiguous()
    if t.is_cuda and torch.cuda.is_current_stream_capturing():
        return v  # a copy made inside a graph capture only holds data once the graph runs
    try:
        t._hxm_f32 = (key, v)
    except (AttributeError, RuntimeError):
        pass
    return v
