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
              mask_b: Tensor | None):
    """sk_row_logprobs on checked, dense arguments: (lse, logprob, entropy,
    top_logprob, top_index, stats); logprob / top_* are None when not asked for."""
    B, N, M = X.shape
    dev = X.device

    def new(*shape, dtype=torch.float32):
        return torch.empty(shape, device=dev, dtype=dtype)

    lse, entropy, stats = new(B, N), new(B, N), new(B, N, 2)
    logprob = new(B, N) if targets is not None else None
    top_lp = new(B, N, top_k) if top_k else None
    top_idx = new(B, N, top_k, dtype=torch.int64) if top_k else None
    if B * N:
        lib = T.lib()
        with torch.cuda.device(dev):
            ws = None if mask_b is None else T.workspace(
                lib.sk_row_logprobs_workspace_bytes(B, M), dev)
            rc = lib.sk_row_logprobs(
                X.data_ptr(), T.DTYPES[X.dtype], B, N, M, *X.stride(), T.ptr(g), epsilon,
                int(negate), T.ptr(mask_a), T.ptr(mask_b), T.ptr(targets), top_k,
                lse.data_ptr(), T.ptr(logprob), entropy.data_ptr(), T.ptr(top_lp),
                T.ptr(top_idx), stats.data_ptr(), T.ptr(ws), 0 if ws is None else ws.numel(),
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

    def dense(t):
        return None if t is None else t.detach().to(torch.float32).contiguous()

    grads = [dense(t) for t in (grad_lse, grad_logprob, grad_entropy, grad_top)]
    if not B * N:
        return dX, None if dg is None else dg.zero_()
    if not (need_dX or need_dg):
        return dX, dg
    lib = T.lib()
    with torch.cuda.device(dev):
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
