"""A mixture of experts routed by balanced optimal transport.

Tokens (rows) and experts (columns) with uniform marginals: the entropic plan gives every
expert the same expected load, whatever the scores favour. ``sinkhorn_route`` solves that
problem and takes each token's best columns under the plan; ``sinkhorn_experts`` runs the
experts' two products on the rows sent to them and sums the results.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Callable

import torch
from torch import Tensor

from . import _tensors as T
from .experts import (MAX_EXPERTS, ExpertDispatch, combine_rows, dispatch_rows,
                      expert_dispatch, grouped_matmul)
from .logprobs import MAX_TOP_K, RowLogprobs, row_logprobs
from .sinkhorn import sinkhorn


@dataclass
class Route:
    """Where each token goes."""

    index: Tensor
    """(T, k) experts of each token, best first; -1 for a masked token"""

    gates: Tensor
    """(T, k) their probabilities under the plan, scaled to sum to 1 per token"""

    dispatch: ExpertDispatch
    """The choices sorted by expert"""

    rows: RowLogprobs
    """lse, entropy and top log probabilities of each token's distribution, (1, T)"""

    n_iters: int
    """Sinkhorn iterations run"""

    converged: bool


def sinkhorn_route(scores: Tensor, top_k: int = 1, epsilon: float = 0.1,
                   mask: Tensor | None = None, max_iters: int = 50, threshold: float = 1e-3,
                   check_every: int = 10) -> Route:
    """Balanced routing of T tokens to E experts by their scores (T, E).

    Solves balanced entropic OT on the cost ``-scores`` (``sinkhorn``, no gradient), then
    takes each token's top_k experts under the plan. The gates are differentiable in the
    scores with the column potential held fixed. mask (T,) bool: tokens that are padding
    go nowhere, and so does a token without a score above -inf (all of them NaN, too: its
    ``rows.lse`` says so). scores float32, bfloat16 or float16; the solve runs in float32
    and waits for its iteration count, as ``sinkhorn`` does.
    """
    if not isinstance(scores, Tensor):
        raise TypeError("scores must be a torch.Tensor")
    if scores.dim() != 2:
        raise ValueError(f"scores must be 2D (T, E), got {scores.dim()}D")
    T.check_dtype(scores, "scores")
    T.check_cuda(scores, "scores")
    t, E = scores.shape
    if t == 0 or E == 0:
        raise ValueError("scores must hold at least one token and one expert")
    if E > MAX_EXPERTS:
        raise ValueError(f"scores must have up to {MAX_EXPERTS} experts, got {E}")
    if not 1 <= top_k <= min(E, MAX_TOP_K):
        raise ValueError(f"top_k must lie between 1 and {min(E, MAX_TOP_K)}, got {top_k}")
    if mask is not None:
        if not isinstance(mask, Tensor):
            raise TypeError("mask must be a torch.Tensor or None")
        if tuple(mask.shape) != (t,):
            raise ValueError(f"mask must have shape {(t,)}, got {tuple(mask.shape)}")
        mask = mask.reshape(1, t)
    C = -scores.to(torch.float32).unsqueeze(0)
    with torch.no_grad():
        out = sinkhorn(C, epsilon=epsilon, mask_a=mask, max_iters=max_iters,
                       threshold=threshold, check_every=check_every)
    rows = row_logprobs(C, out.g, epsilon, top_k=top_k, mask_a=mask)
    index = rows.top_index[0]
    held = index >= 0
    # (a masked token's are all -inf: replaced, so that 0 * nan stays out of the gradient;
    # a NaN among the held ones shows in the gates and in the gradient)
    p = torch.softmax(torch.where(held, rows.top_logprob[0], -1e30), -1)
    gates = torch.where(held, p, torch.zeros_like(p))
    return Route(index, gates, expert_dispatch(index, E), rows, out.n_iters, out.converged)


def sinkhorn_experts(x: Tensor, scores: Tensor, w_in: Tensor, w_out: Tensor, top_k: int = 1,
                     epsilon: float = 0.1,
                     activation: Callable[[Tensor], Tensor] = torch.nn.functional.silu,
                     mask: Tensor | None = None, **solver) -> tuple[Tensor, Route]:
    """A mixture-of-experts feed-forward layer, balanced by optimal transport.

    ``out[t] = sum_j gate[t, j] * activation(x[t] @ w_in[e]) @ w_out[e]`` over token t's
    top_k experts e. x (T, D), w_in (E, D, H), w_out (E, H, D2), all bfloat16 or all
    float16; scores (T, E). Differentiable in x, scores, w_in and w_out. Further arguments
    go to ``sinkhorn_route``. Returns (out, route).
    """
    for name, t, dims in (("x", x, 2), ("scores", scores, 2), ("w_in", w_in, 3),
                          ("w_out", w_out, 3)):
        T.check_cuda(t, name)
        if t.dim() != dims:
            raise ValueError(f"{name} must be {dims}D, got {t.dim()}D")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x is on {x.device}")
        if name != "scores":
            T.check_dtype(t, name, (torch.bfloat16, torch.float16))
            if t.dtype != x.dtype:
                raise TypeError(f"{name} is {t.dtype}, x is {x.dtype}: they must have one type")
    if x.shape[0] != scores.shape[0]:
        raise ValueError(f"x must have {scores.shape[0]} rows, got {x.shape[0]}")
    if w_in.shape[0] != scores.shape[1] or w_out.shape[0] != scores.shape[1]:
        raise ValueError(f"w_in and w_out must hold {scores.shape[1]} experts")
    if w_in.shape[1] != x.shape[1]:
        raise ValueError(f"x has {x.shape[1]} columns, w_in has {w_in.shape[1]} rows")
    route = sinkhorn_route(scores, top_k, epsilon, mask, **solver)
    d = route.dispatch
    h = activation(grouped_matmul(dispatch_rows(x, d), w_in, d.offsets))
    return combine_rows(grouped_matmul(h, w_out, d.offsets), d, route.gates), route
