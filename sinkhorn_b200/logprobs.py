"""Log probabilities of rows, with entropy and the best columns.

A row of the transport plan, normalised, is the distribution
``p_ij = softmax_j((g_j - C_ij) / epsilon)``: which column row i goes to.
``row_logprobs`` gives its log-sum-exp, the log probability of a given column,
its entropy and its k best columns from one read of C (the plan is never
stored); ``token_logprobs`` is the same over logits, as a language model's
output layer has them. Both are differentiable (C or the logits, and g).
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Any

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _tensors as T
from .cuda.row_probs import row_probs, row_probs_backward

MAX_TOP_K = 32


@dataclass
class RowLogprobs:
    """What is known of each row's distribution (fp32; shapes without the column axis)."""

    lse: Tensor
    """log sum exp of the scaled row; -inf for an empty row"""

    entropy: Tensor
    """-sum p log p; 0 for an empty row"""

    logprob: Tensor | None = None
    """log probability of the given column; 0 where none is given (negative
    target), -inf where it is masked, NaN where it is no column"""

    top_logprob: Tensor | None = None
    """log probabilities of the k best columns, descending; -inf where absent"""

    top_index: Tensor | None = None
    """their column numbers (int64), equal values by column; -1 where absent"""


class RowLogprobsFunction(torch.autograd.Function):
    """Autograd wrapper; the backward recomputes p from C and two saved floats a row."""

    @staticmethod
    def forward(ctx: Any, X: Tensor, g: Tensor | None, epsilon: float, negate: bool,
                targets: Tensor | None, top_k: int, mask_a: Tensor | None,
                mask_b: Tensor | None, lead: tuple):
        lse, logprob, entropy, top_lp, top_idx, stats = row_probs(
            X, T.floats(g), epsilon, negate, targets, top_k, mask_a, mask_b, lead, True)
        ctx.set_materialize_grads(False)
        if top_idx is not None:
            ctx.mark_non_differentiable(top_idx)
        ctx.save_for_backward(X, g, targets, mask_b, top_idx, stats, entropy)
        ctx.epsilon = epsilon
        ctx.negate = negate
        return lse, logprob, entropy, top_lp, top_idx

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, g_lse, g_lp, g_ent, g_top, _):
        X, g, targets, mask_b, top_idx, stats, entropy = ctx.saved_tensors
        need_X, need_g = ctx.needs_input_grad[:2]
        if all(t is None for t in (g_lse, g_lp, g_ent, g_top)) or not (need_X or need_g):
            return (None,) * 9
        dX, dg = row_probs_backward(X, T.floats(g), ctx.epsilon, ctx.negate, targets, mask_b,
                                    top_idx, stats, entropy, g_lse, g_lp, g_ent, g_top,
                                    need_X, need_g)
        return (dX, None if dg is None else dg.to(g.dtype)) + (None,) * 7


def _run(X: Tensor, g: Tensor | None, scale: float, negate: bool, targets: Tensor | None,
         top_k: int, mask_a: Tensor | None, mask_b: Tensor | None, lead: tuple):
    if X.stride(2) != 1 and X.shape[2] > 1:
        X = X.contiguous()  # the kernels read rows of unit column stride
    elif X.stride(2) != 1:
        X = X.as_strided(X.shape, (X.stride(0), X.stride(1), 1))
    if T.needs_grad(X, g):
        return RowLogprobsFunction.apply(X, g, scale, negate, targets, top_k, mask_a, mask_b,
                                         lead)
    return row_probs(X, T.floats(g), scale, negate, targets, top_k, mask_a, mask_b, lead,
                     False)[:5]


def _check_top_k(top_k: int, M: int) -> int:
    if isinstance(top_k, bool) or not isinstance(top_k, int):
        raise TypeError("top_k must be an int")
    if not 0 <= top_k <= min(MAX_TOP_K, M):
        raise ValueError(f"top_k must lie between 0 and min({MAX_TOP_K}, columns = {M}), "
                         f"got {top_k}")
    return top_k


def _check_scale(value: float, name: str) -> float:
    value = float(value)
    if not (value > 0 and math.isfinite(value)):
        raise ValueError(f"{name} must be positive and finite, got {value}")
    return value


def row_logprobs(C: Tensor, g: Tensor | None = None, epsilon: float = 0.1,
                 targets: Tensor | None = None, top_k: int = 0,
                 mask_a: Tensor | None = None, mask_b: Tensor | None = None) -> RowLogprobs:
    """The distribution of each row of a transport plan over its columns.

    C (B, N, M) float32, bfloat16 or float16; g (B, M) the column potential (None: 0);
    targets (B, N) integers, one column a row (negative: none); top_k up to 32.
    Rows with ``mask_a`` False, and rows without a column left, are empty; columns with
    ``mask_b`` False have no probability and their C is not looked at (it may be NaN).
    The best columns are those of largest ``g_j - C_ij`` rounded to fp32. Empty rows,
    targets not given, out of range or without probability, absent alternatives and rows
    whose upstream gradients are all zero pass no gradient, whatever such rows hold. All
    arithmetic is fp32; the gradient of C is rounded once to C's type.
    A wait inside the kernel that gives up shows as NaN, not as an error.
    For the distribution of a column over the rows pass ``C.transpose(1, 2)`` and f.
    """
    if not isinstance(C, Tensor):
        raise TypeError("C must be a torch.Tensor")
    if C.dim() != 3:
        raise ValueError(f"C must be 3D (B, N, M), got {C.dim()}D")
    T.check_dtype(C, "C")
    T.check_cuda(C, "C")
    B, N, M = C.shape
    if M == 0:
        raise ValueError("C has no columns")
    top_k = _check_top_k(top_k, M)
    epsilon = _check_scale(epsilon, "epsilon")
    if g is not None:
        if not isinstance(g, Tensor):
            raise TypeError("g must be a torch.Tensor or None")
        if tuple(g.shape) != (B, M):
            raise ValueError(f"g must have shape {(B, M)}, got {tuple(g.shape)}")
        if g.device != C.device:
            raise ValueError(f"g is on {g.device}, C is on {C.device}")
        if not g.dtype.is_floating_point:
            raise TypeError(f"g must be a floating point tensor, got {g.dtype}")
    if targets is not None:
        targets = T.indices(targets, (B, N), C.device, "targets")
    ma = T.mask(mask_a, (B, N), C.device, "mask_a")
    mb = T.mask(mask_b, (B, M), C.device, "mask_b")
    lse, logprob, entropy, top_lp, top_idx = _run(C, g, epsilon, True, targets, top_k, ma, mb,
                                                  (B, N))
    return RowLogprobs(lse, entropy, logprob, top_lp, top_idx)


def token_logprobs(logits: Tensor, targets: Tensor | None = None, top_k: int = 0,
                   temperature: float = 1.0) -> RowLogprobs:
    """Log probabilities of given tokens, entropy and the best alternatives of
    ``softmax(logits / temperature)``.

    logits (..., V) float32, bfloat16 or float16 (rows may be strided); targets (...)
    integers (negative: no token, log probability 0 and no gradient; V or more: NaN);
    top_k up to 32. Logits of -inf have no probability. Gradients as in ``row_logprobs``.
    """
    if not isinstance(logits, Tensor):
        raise TypeError("logits must be a torch.Tensor")
    if logits.dim() < 1:
        raise ValueError("logits must have a vocabulary axis")
    T.check_dtype(logits, "logits")
    T.check_cuda(logits, "logits")
    lead, V = tuple(logits.shape[:-1]), logits.shape[-1]
    if V == 0:
        raise ValueError("logits have an empty vocabulary axis")
    top_k = _check_top_k(top_k, V)
    temperature = _check_scale(temperature, "temperature")
    if targets is not None:
        targets = T.indices(targets, lead, logits.device, "targets")
    if logits.dim() == 3:
        X = logits
    elif logits.dim() == 2:
        X = logits.unsqueeze(0)
    else:
        X = logits.reshape(1, math.prod(lead), V)
    lse, logprob, entropy, top_lp, top_idx = _run(X, None, temperature, False, targets, top_k,
                                                  None, None, lead)
    return RowLogprobs(lse, entropy, logprob, top_lp, top_idx)
