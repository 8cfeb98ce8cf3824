"""Row distributions on the GPU (C ABI wrappers): log-sum-exp, log probability
of a given column, entropy and the best columns of each row in one read of the
cost, and their gradients. ``sinkhorn_b200.logprobs`` is the differentiable
front end.
"""

from __future__ import annotations

import torch
from torch import Tensor

from .. import _tensors as T


def row_probs(X: Tensor, g: Tensor | None, epsilon: float, negate: bool,
              targets: Tensor | None, top_k: int, mask_a: Tensor | None,
              mask_b: Tensor | None, lead: tuple, keep: bool):
    """sk_row_logprobs on checked, dense arguments: (lse, logprob, entropy,
    top_logprob, top_index, stats), of shape ``lead`` (B * N rows); logprob / top_*
    are None when not asked for, stats (for the backward) unless ``keep``."""
    B, N, M = X.shape
    dev = X.device
    f32 = torch.float32
    lse = torch.empty(lead, device=dev, dtype=f32)
    entropy = torch.empty_like(lse)
    stats = torch.empty((B, N, 2), device=dev, dtype=f32) if keep else None
    logprob = torch.empty_like(lse) if targets is not None else None
    top_lp = top_idx = None
    if top_k:
        top_lp = torch.empty((*lead, top_k), device=dev, dtype=f32)
        top_idx = torch.empty((*lead, top_k), device=dev, dtype=torch.int64)
    if B * N:
        lib = T.lib()
        with T.on(dev):
            need = 0 if mask_b is None else lib.sk_row_logprobs_workspace_bytes(B, M)
            ws = T.workspace(need, dev) if need else None
            rc = lib.sk_row_logprobs(
                X.data_ptr(), T.DTYPES[X.dtype], B, N, M, *X.stride(), T.ptr(g), epsilon,
                int(negate), T.ptr(mask_a), T.ptr(mask_b), T.ptr(targets), top_k,
                lse.data_ptr(), T.ptr(logprob), entropy.data_ptr(), T.ptr(top_lp),
                T.ptr(top_idx), T.ptr(stats), T.ptr(ws), 0 if ws is None else ws.numel(),
                T.stream_of(dev))
            T.check(rc, "sk_row_logprobs")
    return lse, logprob, entropy, top_lp, top_idx, stats


def row_probs_backward(X: Tensor, g: Tensor | None, epsilon: float, negate: bool,
                       targets: Tensor | None, mask_b: Tensor | None,
                       top_index: Tensor | None, stats: Tensor, entropy: Tensor,
                       grad_lse: Tensor | None, grad_logprob: Tensor | None,
                       grad_entropy: Tensor | None, grad_top: Tensor | None,
                       need_dX: bool = True, need_dg: bool = True):
    """sk_row_logprobs_backward: (dX, dg); unneeded outputs are None."""
    B, N, M = X.shape
    dev = X.device
    dX = torch.empty(B, N, M, device=dev, dtype=X.dtype) if need_dX else None
    dg = torch.empty(B, M, device=dev, dtype=torch.float32) if need_dg else None

    grads = [T.floats(t) for t in (grad_lse, grad_logprob, grad_entropy, grad_top)]
    if not B * N:
        return dX, None if dg is None else dg.zero_()
    if not (need_dX or need_dg):
        return dX, dg
    lib = T.lib()
    with T.on(dev):
        ws = T.workspace(lib.sk_row_logprobs_backward_workspace_bytes(B, N, M), dev) \
            if need_dg or mask_b is not None else None
        rc = lib.sk_row_logprobs_backward(
            X.data_ptr(), T.DTYPES[X.dtype], B, N, M, *X.stride(), T.ptr(g), epsilon,
            int(negate), T.ptr(mask_b), T.ptr(targets),
            0 if top_index is None else top_index.shape[-1], T.ptr(top_index),
            stats.data_ptr(), entropy.data_ptr(), *(T.ptr(t) for t in grads), T.ptr(dX),
            T.ptr(dg), T.ptr(ws), 0 if ws is None else ws.numel(), T.stream_of(dev))
        T.check(rc, "sk_row_logprobs_backward")
    return dX, dg
