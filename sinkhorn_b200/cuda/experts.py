"""Rows into the order of their experts and back (C ABI wrappers): the stable
sort of a router's choices, the copy of token rows into it, their weighted sum
and its adjoint; and the experts' products over ragged runs of rows. ``sinkhorn_b200.experts`` is the differentiable front end.
"""

from __future__ import annotations

import torch
from torch import Tensor

from .. import _tensors as T


def sort_slots(index: Tensor, n_experts: int) -> tuple[Tensor, Tensor, Tensor]:
    """sk_expert_dispatch on a dense int64 index (T, k): (order, position, offsets)."""
    dev, slots = index.device, index.numel()
    position = torch.empty(index.shape, device=dev, dtype=torch.int32)
    order = position.new_empty(slots)
    if not slots:
        return order, position, torch.zeros(n_experts + 1, device=dev, dtype=torch.int32)
    offsets = position.new_empty(n_experts + 1)
    lib = T.lib()
    with T.on(dev):
        need = lib.sk_expert_dispatch_workspace_bytes(slots, n_experts)
        ws = T.workspace(need, dev) if need else None
        rc = lib.sk_expert_dispatch(index.data_ptr(), slots, n_experts, order.data_ptr(),
                                    position.data_ptr(), offsets.data_ptr(), T.ptr(ws), need,
                                    T.stream_of(dev))
        T.check(rc, "sk_expert_dispatch")
    return order, position, offsets


def unit_rows(x: Tensor) -> Tensor:
    """x itself where its columns have unit stride, else a dense copy."""
    return x if x.stride(1) == 1 or x.shape[1] == 1 and x.is_contiguous() else x.contiguous()


def gather_rows(x: Tensor, order: Tensor, position: Tensor, offsets: Tensor) -> Tensor:
    """sk_dispatch_plan_rows: rows (T k, D) of x (T, D)."""
    x = unit_rows(x)
    t, k = position.shape
    D = x.shape[1]
    rows = torch.empty(t * k, D, device=x.device, dtype=x.dtype)
    if rows.numel():
        with T.on(x.device):
            rc = T.lib().sk_dispatch_plan_rows(
                x.data_ptr(), T.DTYPES[x.dtype], t, k, D, x.stride(0), order.data_ptr(),
                position.data_ptr(), offsets.data_ptr(), offsets.numel() - 1, rows.data_ptr(),
                T.stream_of(x.device))
            T.check(rc, "sk_dispatch_plan_rows")
    return rows


def sum_rows(y: Tensor, order: Tensor, position: Tensor, offsets: Tensor,
             weights: Tensor | None) -> Tensor:
    """sk_combine_plan_rows: (T, D) from y (T k, D); weights dense float32 (T, k) or None."""
    y = unit_rows(y)
    t, k = position.shape
    D = y.shape[1]
    out = torch.empty(t, D, device=y.device, dtype=y.dtype)
    if not out.numel():
        return out
    if not k:
        return out.zero_()
    with T.on(y.device):
        rc = T.lib().sk_combine_plan_rows(
            y.data_ptr(), T.DTYPES[y.dtype], t, k, D, y.stride(0), order.data_ptr(),
            position.data_ptr(), offsets.data_ptr(), offsets.numel() - 1, T.ptr(weights),
            out.data_ptr(), T.stream_of(y.device))
        T.check(rc, "sk_combine_plan_rows")
    return out


def sum_rows_backward(grad: Tensor, y: Tensor, order: Tensor, position: Tensor,
                      offsets: Tensor, weights: Tensor | None, need_y: bool, need_w: bool):
    """sk_combine_plan_rows_backward: (grad_y, grad_weights); unneeded ones are None."""
    t, k = position.shape
    D = y.shape[1]
    grad = unit_rows(grad)
    y = unit_rows(y)
    dy = torch.empty(t * k, D, device=y.device, dtype=y.dtype) if need_y else None
    dw = torch.empty(t, k, device=y.device, dtype=torch.float32) if need_w else None
    if not t * k or not (need_y or need_w):
        return dy, dw
    if not D:
        return dy, None if dw is None else dw.zero_()
    with T.on(y.device):
        rc = T.lib().sk_combine_plan_rows_backward(
            grad.data_ptr(), y.data_ptr(), T.DTYPES[y.dtype], t, k, D, grad.stride(0),
            y.stride(0), order.data_ptr(), position.data_ptr(), offsets.data_ptr(),
            offsets.numel() - 1, T.ptr(weights), T.ptr(dy), T.ptr(dw), T.stream_of(y.device))
        T.check(rc, "sk_combine_plan_rows_backward")
    return dy, dw


def _strides(t: Tensor) -> tuple:
    """Strides of t; an axis of one element has stride 1."""
    if 1 not in t.shape:
        return t.stride()
    return tuple(s if n > 1 else 1 for s, n in zip(t.stride(), t.shape))


def _on_grid(t: Tensor, *strides: int) -> bool:
    return t.data_ptr() % 16 == 0 and all(s % 8 == 0 and s >= 8 for s in strides)


def _packed(t: Tensor, sg: int, sr: int) -> Tensor:
    """sk_grouped_pack: t (groups, rows, width), unit column stride, with rows on 16
    bytes; a view of its width."""
    groups, rows, width = t.shape
    dst = torch.empty(groups, rows, (width + 7) // 8 * 8, device=t.device, dtype=t.dtype)
    with T.on(t.device):
        rc = T.lib().sk_grouped_pack(t.data_ptr(), groups, rows, width, sg, sr,
                                     dst.data_ptr(), T.stream_of(t.device))
        T.check(rc, "sk_grouped_pack")
    return dst[:, :, :width]


def aligned_rows(x: Tensor) -> Tensor:
    """x (S, K) with unit column stride and every row on 16 bytes: itself or a copy."""
    x = unit_rows(x)
    if not x.numel() or _on_grid(x, *([x.stride(0)] if x.shape[0] > 1 else [])):
        return x
    return _packed(x.unsqueeze(0), 0, x.stride(0))[0]


def aligned_weights(w: Tensor) -> Tensor:
    """w (E, K, N) with one of its last two axes of unit stride and every row of that
    axis on 16 bytes: itself or a copy."""
    se, sk, sn = _strides(w)
    if sk != 1 and sn != 1:
        w = w.contiguous()
        se, sk, sn = _strides(w)
    if sn != 1 or (w.shape[2] == 1 and w.shape[1] > 1 and sk == 1):
        return aligned_weights(w.transpose(1, 2)).transpose(1, 2)
    rows = ([sk] if w.shape[1] > 1 else []) + ([se] if w.shape[0] > 1 else [])
    if not w.numel() or _on_grid(w, *rows):
        return w
    return _packed(w, se, sk)


def product(x: Tensor, w: Tensor, offsets: Tensor) -> Tensor:
    """sk_grouped_matmul: (S, N) from x (S, K) (aligned_rows), w (E, K, N)
    (aligned_weights, or transposed) and offsets."""
    S, K = x.shape
    E, _, N = w.shape
    y = torch.empty(S, N, device=x.device, dtype=x.dtype)
    if not y.numel():
        return y
    if not K:
        return y.zero_()
    se, sk, sn = _strides(w)
    if N == 1 and K > 1 and sk == 1:
        sn = K  # one column a group: its K elements are the row
    with T.on(x.device):
        rc = T.lib().sk_grouped_matmul(
            x.data_ptr(), T.DTYPES[x.dtype], S, K, x.stride(0), w.data_ptr(), E, N, se, sk,
            sn, offsets.data_ptr(), y.data_ptr(), T.stream_of(x.device))
        T.check(rc, "sk_grouped_matmul")
    return y


def weight_product(x: Tensor, dy: Tensor, offsets: Tensor, transposed: bool) -> Tensor:
    """sk_grouped_matmul_weight on aligned_rows: dW (E, K, N), laid out (E, N, K) when
    ``transposed``."""
    S, K = x.shape
    N, E = dy.shape[1], offsets.numel() - 1
    dw = torch.empty((E, N, K) if transposed else (E, K, N), device=x.device, dtype=x.dtype)
    if not S:
        dw.zero_()
    elif dw.numel():
        with T.on(x.device):
            rc = T.lib().sk_grouped_matmul_weight(
                x.data_ptr(), T.DTYPES[x.dtype], S, K, x.stride(0), dy.data_ptr(), N,
                dy.stride(0), offsets.data_ptr(), E, dw.data_ptr(), int(transposed),
                T.stream_of(x.device))
            T.check(rc, "sk_grouped_matmul_weight")
    return dw.transpose(1, 2) if transposed else dw
