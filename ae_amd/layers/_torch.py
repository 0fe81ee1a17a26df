"""Torch plumbing for the C ABI: dtype codes, raw pointers, the current HIP stream."""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from .. import _lib

_DTYPE_CODE = {
    torch.float32: _lib.SMX_F32,
    torch.float16: _lib.SMX_F16,
    torch.bfloat16: _lib.SMX_BF16,
}


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _DTYPE_CODE[dt]
    except KeyError:
        raise TypeError(f"unsupported dtype {dt}; expected float32, float16 or bfloat16") from None


def ptr(t: torch.Tensor | None) -> ctypes.c_void_p:
    return ctypes.c_void_p(t.data_ptr() if t is not None else 0)


def stream_of(t: torch.Tensor) -> ctypes.c_void_p:
    """The current torch stream of t's device, as a hipStream_t."""
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def require_gpu(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is not None and t.device.type != "cuda":
            raise ValueError(f"expected a GPU tensor, got one on {t.device}")


def workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    """Per-call scratch from torch's caching allocator (reused across calls, no hipMalloc)."""
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)


raw_stream = torch._C._cuda_getCurrentRawStream  # of a device index: the hipStream_t itself


def rows_of(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """t as a matrix of rows with adjacent elements, and their distance (a copy where needed)."""
    n = t.shape[-1]
    if t.is_contiguous():
        return t, n
    m = t if t.dim() == 2 else t.reshape(-1, n)
    if (m.stride(1) != 1 and n != 1) or (m.stride(0) < n and m.shape[0] > 1):
        m = m.contiguous()
    return m, (m.stride(0) if m.shape[0] > 1 else n)


def address(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def dense(t: torch.Tensor | None) -> torch.Tensor | None:
    return t if t is None or t.is_contiguous() else t.contiguous()


def empty_rows(t: torch.Tensor) -> torch.Tensor:
    """A dense tensor of t's shape and type (empty_like costs half of empty on the host, but keeps other layouts)."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def records_gradient(*tensors: torch.Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def no_tangents(name: str, *tensors: torch.Tensor | None) -> None:
    """Refuses forward-mode duals, whose tangents the kernels would drop."""
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{name} has no forward-mode derivative")


def once(name: str, make, deps, *args) -> tuple:
    """make(*args), the gradients. Where a graph of the gradients themselves is recorded, they depend on deps in a way
    that it cannot differentiate, and says so if it comes to that."""
    if not torch.is_grad_enabled():
        return make(*args)
    with torch.no_grad():
        grads = make(*args)
    deps = [t for t in deps if t is not None]
    return tuple(None if g is None else _Once.apply(name, g, *deps) for g in grads)


class _Once(torch.autograd.Function):
    @staticmethod
    def forward(ctx, name, grad, *deps):
        ctx.name = name
        return grad

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.name} is differentiable once")
