"""Argument checks and pointer plumbing between torch tensors and the C ABI."""

from __future__ import annotations

import contextlib
import math

import torch
from torch import Tensor

from . import _lib


def ptr(t: Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# the handle of a device's current stream without building a Stream object
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_of(device: torch.device) -> int:
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


_HERE = contextlib.nullcontext()


def on(device: torch.device):
    """The device as the current one; nothing to do where it is already."""
    if device.index == torch.cuda.current_device():
        return _HERE
    return torch.cuda.device(device)


def needs_grad(*xs) -> bool:
    return torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in xs)


def tau_arg(tau: float | None) -> float:
    """The C ABI encodes the reference's tau=None (balanced) as +inf."""
    return math.inf if tau is None else float(tau)


def check_cost(C: Tensor, name: str = "C", allow_bf16: bool = False) -> None:
    """allow_bf16: the forward solve also takes a bfloat16 cost (sk_forward_bf16)."""
    if not isinstance(C, Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if C.dim() != 3:
        raise ValueError(f"{name} must be 3D (B, N, M), got {C.dim()}D")
    if not C.is_cuda:
        raise RuntimeError(
            f"{name} is on {C.device}: the cuda backend runs on CUDA tensors only "
            "(there is no CPU fallback)")
    if C.dtype != torch.float32 and not (allow_bf16 and C.dtype == torch.bfloat16):
        raise TypeError(f"{name} must be float32 (the cuda backend computes in fp32"
                        f"{'; the forward solve also takes bfloat16' if allow_bf16 else ''}), "
                        f"got {C.dtype}")
    if any(s < 0 for s in C.stride()):
        raise ValueError(f"{name} has a negative stride")


def vec(x: Tensor | None, shape: tuple, device, name: str) -> Tensor | None:
    """A dense float32 (B,n) vector on `device` (None passes through)."""
    if x is None:
        return None
    if not isinstance(x, Tensor):
        raise TypeError(f"{name} must be a torch.Tensor or None")
    if tuple(x.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, C is on {device}")
    return x.detach().to(torch.float32).contiguous()


def mask(x: Tensor | None, shape: tuple, device, name: str) -> Tensor | None:
    """A dense uint8 (B,n) mask (nonzero = valid)."""
    if x is None:
        return None
    if not isinstance(x, Tensor):
        raise TypeError(f"{name} must be a torch.Tensor or None")
    if tuple(x.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, C is on {device}")
    if x.dtype == torch.bool:
        return x.contiguous().view(torch.uint8)
    return (x != 0).contiguous().view(torch.uint8)


# element types of the operators that take more than float32 (sk_dtype)
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def check_cuda(x: Tensor, name: str) -> None:
    if not isinstance(x, Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not x.is_cuda:
        raise RuntimeError(f"{name} is on {x.device}: the cuda backend runs on CUDA tensors "
                           "only (there is no CPU fallback)")


def check_dtype(x: Tensor, name: str, allowed=tuple(DTYPES)) -> None:
    if x.dtype not in allowed:
        names = ", ".join(str(d).replace("torch.", "") for d in allowed)
        raise TypeError(f"{name} must be one of {names}, got {x.dtype}")


def indices(x: Tensor, shape: tuple, device, name: str) -> Tensor:
    """A dense int64 tensor of `shape` on `device` from any integer type."""
    if not isinstance(x, Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if x.dtype not in (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8):
        raise TypeError(f"{name} must hold integers, got {x.dtype}")
    if tuple(x.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, expected {device}")
    if x.dtype == torch.int64 and x.is_contiguous():
        return x
    return x.to(torch.int64).contiguous()


def floats(x: Tensor | None) -> Tensor | None:
    """A dense float32 tensor outside the autograd graph (None passes through)."""
    if x is None:
        return None
    x = x.detach()
    return x if x.dtype == torch.float32 and x.is_contiguous() \
        else x.to(torch.float32).contiguous()


def workspace(nbytes: int, device) -> Tensor:
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


def cost_args(C: Tensor) -> tuple:
    B, N, M = C.shape
    sb, sn, sm = C.stride()
    return (C.data_ptr(), B, N, M, sb, sn, sm)


lib = _lib.load
check = _lib.check
