"""Rows to experts and back, next to a Sinkhorn router.

A router (a transport plan's best columns, ``row_logprobs(..., top_k=k)``) gives each
token k experts. ``expert_dispatch`` sorts these choices by expert, ``dispatch_rows``
copies the tokens' rows into that order, so that each expert's rows are consecutive,
``grouped_matmul`` multiplies them by their experts' weights, and ``combine_rows`` sums each
token's k results with its gates. All but the sort are differentiable; nothing here
synchronises with the host.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Any

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _tensors as T
from .cuda.experts import (aligned_rows, aligned_weights, gather_rows, product, sort_slots,
                           sum_rows, sum_rows_backward, weight_product)

MAX_EXPERTS = 1024


@dataclass
class ExpertDispatch:
    """Where each slot (token t's j-th choice, number t * k + j) goes. int32 tensors.

    A slot holds place ``position[t, j]`` where ``order`` names the slot there and the place
    lies before the last offset; any other slot counts as dropped, and a place that no slot
    holds is a row of zeros. So a plan may be edited, as for experts over their capacity:
    -1 in ``position`` drops a slot."""

    order: Tensor
    """(T k,) the slot at each place, -1 behind the last group"""

    position: Tensor
    """(T, k) the place of each slot, -1 for a choice that is no expert"""

    offsets: Tensor
    """(E + 1,) first place of each expert's group; the last entry ends them all"""

    @property
    def n_experts(self) -> int:
        return self.offsets.numel() - 1


def expert_dispatch(index: Tensor, n_experts: int) -> ExpertDispatch:
    """Sort the choices index (T, k) (integers) by expert, equal ones by slot.

    Choices outside 0..n_experts-1 (-1, as ``row_logprobs`` gives for rows without
    a column) are dropped. Up to 1024 experts.
    """
    if not isinstance(index, Tensor):
        raise TypeError("index must be a torch.Tensor")
    if index.dim() != 2:
        raise ValueError(f"index must be 2D (T, k), got {index.dim()}D")
    if isinstance(n_experts, bool) or not isinstance(n_experts, int):
        raise TypeError("n_experts must be an int")
    if not 1 <= n_experts <= MAX_EXPERTS:
        raise ValueError(f"n_experts must lie between 1 and {MAX_EXPERTS}, got {n_experts}")
    if index.numel() >= 2 ** 31:
        raise ValueError("index must have fewer than 2^31 entries")
    T.check_cuda(index, "index")
    index = T.indices(index, index.shape, index.device, "index")
    return ExpertDispatch(*sort_slots(index, n_experts))


def _check_dispatch(d: ExpertDispatch, device) -> None:
    if not isinstance(d, ExpertDispatch):
        raise TypeError("dispatch must be an ExpertDispatch")
    for name in ("order", "position", "offsets"):
        t = getattr(d, name)
        if not isinstance(t, Tensor) or t.dtype != torch.int32:
            raise TypeError(f"dispatch.{name} must be an int32 tensor")
        if t.device != device:
            raise ValueError(f"dispatch.{name} is on {t.device}, the rows are on {device}")
        if not t.is_contiguous():
            raise ValueError(f"dispatch.{name} must be contiguous")
    if d.position.dim() != 2 or d.order.shape != (d.position.numel(),):
        raise ValueError("dispatch.position must be (T, k) and dispatch.order (T k,)")
    if d.offsets.dim() != 1 or not 2 <= d.offsets.numel() <= MAX_EXPERTS + 1:
        raise ValueError(f"dispatch.offsets must have 2 to {MAX_EXPERTS + 1} entries")


def _check_rows(x: Tensor, name: str, rows: int) -> None:
    if x.dim() != 2:
        raise ValueError(f"{name} must be 2D, got {x.dim()}D")
    T.check_dtype(x, name)
    if x.shape[0] != rows:
        raise ValueError(f"{name} must have {rows} rows, got {x.shape[0]}")


class DispatchRowsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: Tensor, order: Tensor, position: Tensor,
                offsets: Tensor) -> Tensor:
        ctx.save_for_backward(order, position, offsets)
        return gather_rows(x, order, position, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad: Tensor):
        return sum_rows(grad, *ctx.saved_tensors, None), None, None, None


class CombineRowsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, y: Tensor, weights: Tensor | None, order: Tensor, position: Tensor,
                offsets: Tensor) -> Tensor:
        ctx.save_for_backward(y, weights, order, position, offsets)
        return sum_rows(y, order, position, offsets, T.floats(weights))

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad: Tensor):
        y, weights, order, position, offsets = ctx.saved_tensors
        dy, dw = sum_rows_backward(grad, y, order, position, offsets, T.floats(weights),
                                   ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dy, None if dw is None else dw.to(weights.dtype), None, None, None


def dispatch_rows(x: Tensor, dispatch: ExpertDispatch) -> Tensor:
    """Rows of x (T, D) in expert order: (T k, D), row ``position[t, j]`` is x[t].

    Rows that no slot holds are zero, those behind the last group among them. float32, bfloat16 or float16; rows may be
    strided. The gradient of x[t] is the sum over its rows, in fp32, rounded once.
    """
    T.check_cuda(x, "x")
    _check_dispatch(dispatch, x.device)
    _check_rows(x, "x", dispatch.position.shape[0])
    if not T.needs_grad(x):
        return gather_rows(x, dispatch.order, dispatch.position, dispatch.offsets)
    return DispatchRowsFunction.apply(x, dispatch.order, dispatch.position, dispatch.offsets)


def combine_rows(y: Tensor, dispatch: ExpertDispatch, weights: Tensor | None = None) -> Tensor:
    """``out[t] = sum_j weights[t, j] * y[position[t, j]]`` (T, D): the experts' rows back
    to their tokens.

    y (T k, D) float32, bfloat16 or float16; weights (T, k) floating point, None for 1.
    Dropped choices add nothing and their weights get no gradient. Sums are in fp32.
    """
    T.check_cuda(y, "y")
    _check_dispatch(dispatch, y.device)
    t, k = dispatch.position.shape
    _check_rows(y, "y", t * k)
    if weights is not None:
        if not isinstance(weights, Tensor):
            raise TypeError("weights must be a torch.Tensor or None")
        if not weights.dtype.is_floating_point:
            raise TypeError(f"weights must be floating point, got {weights.dtype}")
        if tuple(weights.shape) != (t, k):
            raise ValueError(f"weights must have shape {(t, k)}, got {tuple(weights.shape)}")
        if weights.device != y.device:
            raise ValueError(f"weights are on {weights.device}, y is on {y.device}")
    if not T.needs_grad(y, weights):
        return sum_rows(y, dispatch.order, dispatch.position, dispatch.offsets,
                        T.floats(weights))
    return CombineRowsFunction.apply(y, weights, dispatch.order, dispatch.position,
                                     dispatch.offsets)


class GroupedMatmulFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: Tensor, w: Tensor, offsets: Tensor) -> Tensor:
        x, w = aligned_rows(x), aligned_weights(w)
        ctx.save_for_backward(x, w, offsets)
        ctx.transposed = w.stride(2) != 1 and w.shape[2] > 1
        return product(x, w, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad: Tensor):
        x, w, offsets = ctx.saved_tensors
        dx = dw = None
        grad = aligned_rows(grad)
        if ctx.needs_input_grad[0]:
            dx = product(grad, w.transpose(1, 2), offsets)
        if ctx.needs_input_grad[1]:
            dw = weight_product(x, grad, offsets, ctx.transposed)
        return dx, dw, None


def grouped_matmul(x: Tensor, w: Tensor, offsets: Tensor) -> Tensor:
    """``y[r] = x[r] @ w[e]`` for the rows r of each group e: (S, N).

    x (S, K) and w (E, K, N), both bfloat16 or both float16; offsets (E + 1,) int32 or
    int64 on the device, group e holds rows ``offsets[e]`` to ``offsets[e + 1] - 1`` (as
    ``expert_dispatch`` gives them). Groups may be empty; rows of no group give zeros and
    get zero gradient. Offsets that decrease or leave 0..S are clamped. Sums are in fp32,
    rounded once. Any K and N; rows that do not start on 16 bytes (K or N no multiple of 8)
    are copied once more. w may be stored (E, N, K) and passed transposed; its gradient then
    has that layout, too. Up to 1024 groups. A wait inside the kernel that gives up shows as
    NaN in the output, not as an error: nothing here waits for the device.
    """
    for name, t, dims in (("x", x, 2), ("w", w, 3)):
        T.check_cuda(t, name)
        if t.dim() != dims:
            raise ValueError(f"{name} must be {dims}D, got {t.dim()}D")
        T.check_dtype(t, name, (torch.bfloat16, torch.float16))
    if x.dtype != w.dtype:
        raise TypeError(f"x is {x.dtype}, w is {w.dtype}: they must have one type")
    if w.device != x.device:
        raise ValueError(f"w is on {w.device}, x is on {x.device}")
    E, K, _ = w.shape
    if x.shape[1] != K:
        raise ValueError(f"x has {x.shape[1]} columns, w has {K} rows")
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"w must hold 1 to {MAX_EXPERTS} groups, got {E}")
    if not isinstance(offsets, Tensor):
        raise TypeError("offsets must be a torch.Tensor")
    if offsets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"offsets must be int32 or int64, got {offsets.dtype}")
    if tuple(offsets.shape) != (E + 1,):
        raise ValueError(f"offsets must have shape {(E + 1,)}, got {tuple(offsets.shape)}")
    if offsets.device != x.device:
        raise ValueError(f"offsets are on {offsets.device}, x is on {x.device}")
    if offsets.dtype == torch.int64:
        offsets = offsets.clamp(0, x.shape[0]).to(torch.int32)
    offsets = offsets.contiguous()
    if not T.needs_grad(x, w):
        return product(aligned_rows(x), aligned_weights(w), offsets)
    return GroupedMatmulFunction.apply(x, w, offsets)
