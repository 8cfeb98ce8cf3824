"""Cases of the operators around a Sinkhorn router and a model's output rows.

Three operators, each in the forms that serving and training call:

* row / token log probabilities with entropy and top alternatives (``row_logprobs`` over a cost and a column
  potential, ``token_logprobs`` over logits), with their gradients;
* ``expert_dispatch`` / ``dispatch_rows`` / ``combine_rows``: rows into expert order and back, with gradients;
* ``grouped_matmul``: the experts' products over ragged groups of rows, with both gradients.

``run`` computes a case in elementary torch operations; with ``own`` set it calls sinkhorn_b200 instead.
``exact`` computes it again from the definitions in 64 bits.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one sequence's new token: log probability, entropy and 20 alternatives for the client
        {"name": "logprobs-decode", "op": "logprobs", "rows": 1, "vocab": 131072, "dtype": "bf16", "top": 20, "temperature": 0.8},
        # prompt log probabilities of a packed batch, an odd vocabulary
        {"name": "logprobs-prompt", "op": "logprobs", "rows": 4096, "vocab": 50001, "dtype": "bf16", "top": 5, "temperature": 1.0},
        # policy-gradient step: log probabilities and entropy with the gradient of the logits
        {"name": "logprobs-train", "op": "logprobs_train", "rows": 8192, "vocab": 65536, "dtype": "bf16", "top": 0, "temperature": 1.0},
        # best matches of each row of a batch of transport problems, some columns masked
        {"name": "plan-rows", "op": "plan_rows", "batch": 16, "rows": 2048, "cols": 2048, "top": 4, "epsilon": 0.05, "masked": True},
        # router of a training step: two experts a token, gradients of the scores and of the column potential
        {"name": "router-train", "op": "plan_rows_train", "batch": 4, "rows": 8192, "cols": 64, "top": 2, "epsilon": 0.05, "masked": False},
        # a small decoding batch into expert order
        {"name": "dispatch-decode", "op": "dispatch", "tokens": 100, "top": 2, "experts": 64, "width": 2048, "dtype": "bf16"},
        # a training batch into expert order
        {"name": "dispatch-batch", "op": "dispatch", "tokens": 32768, "top": 2, "experts": 128, "width": 2048, "dtype": "bf16"},
        # the experts' rows back to the tokens, with the gradients of the rows and of the gates; odd token count
        {"name": "combine-train", "op": "combine_train", "tokens": 16385, "top": 4, "experts": 64, "width": 1536, "dtype": "bf16"},
        # experts of a small decoding batch: bound by the read of the weights
        {"name": "experts-decode", "op": "grouped", "rows": 200, "experts": 64, "k": 2048, "n": 1024, "dtype": "bf16"},
        # experts of a prompt batch
        {"name": "experts-prompt", "op": "grouped", "rows": 16384, "experts": 16, "k": 2048, "n": 4096, "dtype": "bf16"},
        # experts of a training step, forward and both gradients
        {"name": "experts-train", "op": "grouped_train", "rows": 16384, "experts": 8, "k": 4096, "n": 2048, "dtype": "bf16"},
        # odd widths, half precision, forward and both gradients
        {"name": "experts-odd", "op": "grouped_train", "rows": 5003, "experts": 5, "k": 1001, "n": 777, "dtype": "fp16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "logprobs_train", "plan_rows", "plan_rows_train", "dispatch", "combine_train",
                     "grouped", "grouped", "grouped_train"])
    if op in ("logprobs", "logprobs_train"):
        vocab = _log_int(rng, 500, 200000)
        most = max(1, min(16384, (8192 * 65536) // vocab))
        return {"op": op, "rows": _log_int(rng, 1, most), "vocab": vocab, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "top": 0 if op == "logprobs_train" else rng.choice([0, 1, 5, 20, 32]), "temperature": rng.choice([0.7, 1.0, 1.3])}
    if op in ("plan_rows", "plan_rows_train"):
        cols = _log_int(rng, 4, 4096)
        batch = rng.randint(1, 8)
        most = max(1, min(16384, (16 * 2048 * 2048) // (cols * batch)))
        return {"op": op, "batch": batch, "rows": _log_int(rng, 1, most), "cols": cols, "top": rng.randint(1, min(8, cols)),
                "epsilon": rng.choice([0.05, 0.1, 1.0]), "masked": rng.random() < 0.5}
    if op in ("dispatch", "combine_train"):
        return {"op": op, "tokens": _log_int(rng, 1, 16384), "top": rng.randint(1, 4), "experts": _log_int(rng, 4, 256),
                "width": rng.choice([_log_int(rng, 64, 2048), 8 * _log_int(rng, 8, 256)]), "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    widths = [rng.choice([_log_int(rng, 64, 4096), 8 * _log_int(rng, 8, 512), 8 * _log_int(rng, 8, 512)]) for _ in range(2)]
    return {"op": op, "rows": _log_int(rng, 1, 8192), "experts": _log_int(rng, 1, 64), "k": widths[0], "n": widths[1] // 2 + 32,
            "dtype": rng.choice(["bf16", "fp16"])}


def _scores(gen, rows, cols):
    """Affinities as a router sees them: noise around a popularity of each column."""
    return torch.randn(rows, cols, device="cuda", generator=gen) + 0.5 * torch.randn(cols, device="cuda", generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": case}

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", generator=gen).to(dtype)

    if op in ("logprobs", "logprobs_train"):
        T, V = case["rows"], case["vocab"]
        logits = (2.5 * randn(T, V)).to(_TYPES[case["dtype"]])
        s["targets"] = torch.randint(0, V, (T,), device="cuda", generator=gen)
        if op == "logprobs_train":
            # the last position of a padded batch has no token
            s["targets"][-1:] = -100 if T > 1 else s["targets"][-1]
            s["grads"] = (randn(T) / T, 0.01 * randn(T) / T)
        s["logits"] = logits.requires_grad_(op == "logprobs_train")
    elif op in ("plan_rows", "plan_rows_train"):
        B, N, M = case["batch"], case["rows"], case["cols"]
        train = op == "plan_rows_train"
        s["C"] = (-_scores(gen, B * N, M)).view(B, N, M).requires_grad_(train)
        s["g"] = (0.3 * randn(B, M)).requires_grad_(train)
        s["mask_b"] = None
        if case["masked"]:
            mask = torch.rand(B, M, device="cuda", generator=gen) > 0.1
            mask[:, -1] = True
            s["mask_b"] = mask
        if train:
            s["grads"] = (randn(B, N) / N, randn(B, N, case["top"]) / N)
    elif op in ("dispatch", "combine_train"):
        T, k, E, D = case["tokens"], case["top"], case["experts"], case["width"]
        index = _scores(gen, T, E).topk(k, dim=1).indices
        # padded tokens go to no expert
        index[torch.rand(T, device="cuda", generator=gen) < 0.02] = -1
        s["index"] = index
        if op == "dispatch":
            s["x"] = randn(T, D, dtype=_TYPES[case["dtype"]])
        else:
            s["y"] = randn(T * k, D, dtype=_TYPES[case["dtype"]]).requires_grad_()
            s["weights"] = torch.rand(T, k, device="cuda", generator=gen).requires_grad_()
            s["grad"] = randn(T, D, dtype=_TYPES[case["dtype"]])
            s["plan"] = _plan(index, E)
    else:
        S, E, K, N = case["rows"], case["experts"], case["k"], case["n"]
        dt = _TYPES[case["dtype"]]
        # ragged lengths: a popularity of each expert, one expert without rows where there are several, a few rows behind the last group
        host = torch.Generator().manual_seed(seed)
        share = torch.softmax(0.5 * torch.randn(E, generator=host), 0)
        if E > 1:
            share[int(torch.randint(0, E, (1,), generator=host))] = 0.0
        used = S - S // 100
        lengths = torch.bincount(torch.multinomial(share, used, replacement=True, generator=host), minlength=E)
        s["longest"] = int(lengths.max())
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)]).to(torch.int32).cuda()
        train = op == "grouped_train"
        s["x"] = randn(S, K, dtype=dt).requires_grad_(train)
        s["w"] = (randn(E, K, N) / math.sqrt(K)).to(dt).requires_grad_(train)
        if train:
            s["grad"] = randn(S, N, dtype=dt)
    return s


# ---------------------------------------------------------------------------------------------- the plain forms


def _descending(x, k):
    """Indices of the k largest of each row, ties to the lowest index, -1 where a row has fewer that are above -inf."""
    bits = (x + 0.0).view(torch.int32)
    ordered = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).to(torch.int64)
    place = torch.arange(x.shape[-1], device=x.device)
    index = torch.topk((ordered << 32) + (0x7FFFFFFF - place), k, dim=-1).indices
    return torch.where(x.gather(-1, index) > -math.inf, index, -1)


def _softmax_parts(x, scale):
    """z, log sum exp, probabilities and entropy of rows x * scale, in 32 bits."""
    z = x * scale
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    lse = torch.log(total) + top
    p = e / total
    logp = z - lse
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    return lse, p, logp, entropy


def _pick(logp, index):
    """logp at index, -inf where the index is -1."""
    return torch.where(index >= 0, logp.gather(-1, index.clamp(min=0)), torch.full_like(logp[..., :1], -math.inf))


def _logits_gradient(p, logp, entropy, scale, gl, targets, gh):
    """(1/temperature) of gl ([v = t] - p) - gh p (log p + H)."""
    given = targets >= 0
    a = torch.where(given, gl, torch.zeros_like(gl))
    d = -p * (a[:, None] + gh[:, None] * torch.where(p > 0, logp + entropy[:, None], torch.zeros_like(p)))
    d.scatter_add_(1, targets.clamp(min=0)[:, None], a[:, None])
    return d * scale


def _plan(index, experts):
    """Stable order of the slots by expert: order, position, offsets."""
    flat = index.reshape(-1)
    valid = (flat >= 0) & (flat < experts)
    key = torch.where(valid, flat, torch.full_like(flat, experts))
    order = torch.sort(key, stable=True).indices
    counts = (key[:, None] == torch.arange(experts, device=key.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    place = torch.arange(flat.numel(), device=flat.device)
    position = torch.empty_like(order)
    position[order] = place
    position = torch.where(valid, position, -1).view(index.shape)
    order = torch.where(place < offsets[-1], order, -1)
    return order.to(torch.int32), position.to(torch.int32), offsets.to(torch.int32)


def _grouped_rows(s):
    """Row numbers of each group padded to the longest, and where they hold."""
    offsets = s["offsets"].long()
    rows = offsets[:-1, None] + torch.arange(s["longest"], device=offsets.device)
    return rows.clamp(max=s["x"].shape[0] - 1), rows < offsets[1:, None]


def _padded(x, rows, holds):
    return torch.where(holds[..., None], x[rows].float(), 0.0)


def _unpadded(y, s, dtype):
    offsets = s["offsets"].long()
    row = torch.arange(s["x"].shape[0], device=y.device)
    group = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
    inside = group < y.shape[0]
    group = torch.where(inside, group, 0)
    local = torch.where(inside, row - offsets[group], 0)
    return torch.where(inside[:, None], y[group, local], 0.0).to(dtype)


@torch.no_grad()
def _run_plain(s):
    case, op = s["case"], s["case"]["op"]
    if op in ("logprobs", "logprobs_train"):
        x = s["logits"].detach().float()
        scale = 1.0 / case["temperature"]
        lse, p, logp, entropy = _softmax_parts(x, scale)
        logprob = torch.where(s["targets"] >= 0, _pick(logp, s["targets"][:, None])[:, 0], 0.0)
        if op == "logprobs_train":
            grad = _logits_gradient(p, logp, entropy, scale, s["grads"][0], s["targets"], s["grads"][1])
            return {"logprob": logprob, "entropy": entropy, "grad": grad.to(s["logits"].dtype)}
        out = {"logprob": logprob, "entropy": entropy}
        if case["top"]:
            out["top_index"] = _descending(x, case["top"])
            out["top_logprob"] = _pick(logp, out["top_index"])
        return out
    if op in ("plan_rows", "plan_rows_train"):
        x = s["g"].detach()[:, None, :] - s["C"].detach()
        if s["mask_b"] is not None:
            x = torch.where(s["mask_b"][:, None, :], x, -math.inf)
        scale = 1.0 / case["epsilon"]
        lse, p, logp, entropy = _softmax_parts(x, scale)
        index = _descending(x, case["top"])
        out = {"entropy": entropy, "top_index": index, "top_logprob": _pick(logp, index)}
        if op == "plan_rows_train":
            gh, gt = s["grads"]
            gt = torch.where(index >= 0, gt, torch.zeros_like(gt))
            d = -p * (gt.sum(-1, keepdim=True) + gh[..., None] * torch.where(p > 0, logp + entropy[..., None], torch.zeros_like(p)))
            d.scatter_add_(-1, index.clamp(min=0), gt)
            d = d * scale
            out["grad_C"], out["grad_g"] = -d, d.sum(1)
        return out
    if op == "dispatch":
        order, position, offsets = _plan(s["index"], case["experts"])
        token = torch.div(order.long().clamp(min=0), case["top"], rounding_mode="floor")
        rows = torch.where(order[:, None] >= 0, s["x"][token], torch.zeros_like(s["x"][:1]))
        return {"order": order, "position": position, "offsets": offsets, "rows": rows}
    if op == "combine_train":
        order, position, _ = s["plan"]
        y, w, grad = s["y"].detach(), s["weights"].detach(), s["grad"].float()
        T, k = position.shape
        at = position.long()
        held = torch.where(at[..., None] >= 0, y[at.clamp(min=0)].float(), 0.0)
        out = (w[..., None] * held).sum(1).to(y.dtype)
        slot = order.long().clamp(min=0)
        dy = torch.where(order[:, None] >= 0, w.reshape(-1)[slot][:, None] * grad[torch.div(slot, k, rounding_mode="floor")], 0.0).to(y.dtype)
        return {"out": out, "grad_y": dy, "grad_weights": (held * grad[:, None, :]).sum(-1)}
    x, w = s["x"].detach(), s["w"].detach()
    rows, holds = _grouped_rows(s)
    xp, wf = _padded(x, rows, holds), w.float()
    out = {"y": _unpadded(torch.bmm(xp, wf), s, x.dtype)}
    if op == "grouped_train":
        gp = _padded(s["grad"], rows, holds)
        out["grad_x"] = _unpadded(torch.bmm(gp, wf.transpose(1, 2)), s, x.dtype)
        out["grad_w"] = torch.bmm(xp.transpose(1, 2), gp).to(w.dtype)
    return out


# ------------------------------------------------------------------------------------- the framework's operators


def _run_own(s):
    import sinkhorn_b200 as skb

    case, op = s["case"], s["case"]["op"]
    if op == "logprobs":
        r = skb.token_logprobs(s["logits"], s["targets"], top_k=case["top"], temperature=case["temperature"])
        out = {"logprob": r.logprob, "entropy": r.entropy}
        if case["top"]:
            out["top_index"], out["top_logprob"] = r.top_index, r.top_logprob
        return out
    if op == "logprobs_train":
        r = skb.token_logprobs(s["logits"], s["targets"], temperature=case["temperature"])
        grad, = torch.autograd.grad((r.logprob, r.entropy), (s["logits"],), s["grads"])
        return {"logprob": r.logprob.detach(), "entropy": r.entropy.detach(), "grad": grad}
    if op in ("plan_rows", "plan_rows_train"):
        r = skb.row_logprobs(s["C"], s["g"], case["epsilon"], top_k=case["top"], mask_b=s["mask_b"])
        out = {"entropy": r.entropy.detach(), "top_index": r.top_index, "top_logprob": r.top_logprob.detach()}
        if op == "plan_rows_train":
            out["grad_C"], out["grad_g"] = torch.autograd.grad((r.entropy, r.top_logprob), (s["C"], s["g"]), s["grads"])
        return out
    if op == "dispatch":
        d = skb.expert_dispatch(s["index"], case["experts"])
        return {"order": d.order, "position": d.position, "offsets": d.offsets, "rows": skb.dispatch_rows(s["x"], d)}
    if op == "combine_train":
        out = skb.combine_rows(s["y"], skb.ExpertDispatch(*s["plan"]), s["weights"])
        dy, dw = torch.autograd.grad(out, (s["y"], s["weights"]), s["grad"])
        return {"out": out.detach(), "grad_y": dy, "grad_weights": dw}
    y = skb.grouped_matmul(s["x"], s["w"], s["offsets"])
    out = {"y": y.detach()}
    if op == "grouped_train":
        out["grad_x"], out["grad_w"] = torch.autograd.grad(y, (s["x"], s["w"]), s["grad"])
    return out


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ------------------------------------------------------------------------------------------------ work and exact


def work(case):
    op = case["op"]
    if op in ("logprobs", "logprobs_train"):
        T, V, b = case["rows"], case["vocab"], _SIZE[case["dtype"]]
        train = op == "logprobs_train"
        bytes_ = T * V * b * (2 if train else 1) + T * (8 + 8 + 12 * case["top"] + (8 if train else 0))
        return {"bytes": bytes_, "flops": T * V * (12 if train else 6)}
    if op in ("plan_rows", "plan_rows_train"):
        B, N, M, k = case["batch"], case["rows"], case["cols"], case["top"]
        train = op == "plan_rows_train"
        bytes_ = B * N * M * 4 * (2 if train else 1) + B * N * (4 + 12 * k) + B * M * 5
        if train:
            bytes_ += B * N * (4 + 4 * k) + B * M * 4
        return {"bytes": bytes_, "flops": B * N * M * (14 if train else 7)}
    if op in ("dispatch", "combine_train"):
        T, k, E, D, b = case["tokens"], case["top"], case["experts"], case["width"], _SIZE[case["dtype"]]
        if op == "dispatch":
            return {"bytes": T * D * b + T * k * (D * b + 8 + 8) + 4 * E, "flops": T * k}
        return {"bytes": 2 * T * k * D * b + 2 * T * D * b + T * k * 16, "flops": 5 * T * k * D}
    S, E, K, N, b = case["rows"], case["experts"], case["k"], case["n"], _SIZE[case["dtype"]]
    # the rows of no group (one in a hundred) cost no products; an expert without rows no weights
    held, used = S - S // 100, max(1, min(E - 1 if E > 1 else 1, S))
    if op == "grouped":
        return {"bytes": b * (held * K + S * N + used * K * N), "flops": 2 * held * K * N}
    # forward: x, w in, y out; gradients: grad in, grad_x and grad_w out
    return {"bytes": b * (held * K + S * N + used * K * N) + b * (held * N + S * K + E * K * N), "flops": 6 * held * K * N}


def _exact_rows(x64, x32, scale, top):
    z = x64 * scale
    lse = torch.logsumexp(z, -1, keepdim=True)
    lp = torch.where(torch.isinf(lse), torch.full_like(z, -math.inf), z - lse)
    p = torch.exp(lp)
    h = -(torch.where(p > 0, lp, 0.0) * p).sum(-1)
    index = None
    if top:
        # the order is that of the 32-bit values, equal ones by their place
        index = torch.sort(x32, dim=-1, descending=True, stable=True).indices[..., :top]
        index = torch.where(torch.isinf(x32.gather(-1, index)), -1, index)
    return lp, p, h, index


def _at(lp, index):
    return torch.where(index >= 0, lp.gather(-1, index.clamp(min=0)), -math.inf)


@torch.no_grad()
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op in ("logprobs", "logprobs_train"):
        T, t = case["rows"], s["targets"]
        step = max(1, (1 << 27) // case["vocab"])
        parts = []
        for r in range(0, T, step):
            x32 = s["logits"].detach()[r:r + step].float()
            lp, p, h, index = _exact_rows(x32.double(), x32, 1.0 / case["temperature"], case["top"])
            tr = t[r:r + step]
            got = {"logprob": torch.where(tr >= 0, lp.gather(1, tr.clamp(min=0)[:, None])[:, 0], 0.0), "entropy": h}
            if case["top"]:
                got["top_logprob"] = _at(lp, index)
            if op == "logprobs_train":
                gl, gh = s["grads"][0][r:r + step].double(), s["grads"][1][r:r + step].double()
                one = torch.zeros_like(p)
                one.scatter_(1, tr.clamp(min=0)[:, None], 1.0)
                a = torch.where(tr >= 0, gl, 0.0)[:, None]
                got["grad"] = (a * (one - p) - gh[:, None] * p * (torch.where(p > 0, lp, 0.0) + h[:, None])) / case["temperature"]
            parts.append(got)
        out = {k: torch.cat([q[k] for q in parts]) for k in parts[0]}
        if op == "logprobs_train":
            return {"logprob": out["logprob"], "entropy": out["entropy"], "grad": out["grad"]}
        if case["top"]:
            return {"logprob": out["logprob"], "entropy": out["entropy"], "top_index": None, "top_logprob": out["top_logprob"]}
        return out
    if op in ("plan_rows", "plan_rows_train"):
        C, g, m = s["C"].detach(), s["g"].detach(), s["mask_b"]
        x32, x64 = g[:, None] - C, g.double()[:, None] - C.double()
        if m is not None:
            x32, x64 = x32.masked_fill(~m[:, None], -math.inf), x64.masked_fill(~m[:, None], -math.inf)
        lp, p, h, index = _exact_rows(x64, x32, 1.0 / case["epsilon"], case["top"])
        out = {"entropy": h, "top_index": None, "top_logprob": _at(lp, index)}
        if op == "plan_rows_train":
            gh, gt = s["grads"][0].double(), s["grads"][1].double()
            gt = gt * (index >= 0)
            dz = -p * gt.sum(-1, keepdim=True) - gh[..., None] * p * (torch.where(p > 0, lp, 0.0) + h[..., None])
            dz = dz.scatter_add(-1, index.clamp(min=0), gt) / case["epsilon"]
            out["grad_C"], out["grad_g"] = -dz, dz.sum(1)
        return out
    if op == "dispatch":
        flat = s["index"].reshape(-1)
        order = torch.sort(torch.where(flat < 0, case["experts"], flat), stable=True).indices
        rows = s["x"].double()[order // case["top"]] * (flat[order] >= 0)[:, None]
        return {"order": None, "position": None, "offsets": None, "rows": rows}
    if op == "combine_train":
        order = torch.sort(torch.where(s["index"] < 0, case["experts"], s["index"]).reshape(-1), stable=True).indices
        T, k = s["index"].shape
        y, w, d = s["y"].detach().double(), s["weights"].detach().double(), s["grad"].double()
        w = w * (s["index"] >= 0)
        by_slot = torch.empty_like(y)
        by_slot[order] = y
        by_slot = by_slot.view(T, k, -1)
        dy = (w[..., None] * d[:, None]).reshape(T * k, -1)[order]
        return {"out": torch.einsum("tk,tkd->td", w, by_slot), "grad_y": dy,
                "grad_weights": torch.einsum("td,tkd->tk", d, by_slot) * (s["index"] >= 0)}
    x, w, ends = s["x"].detach().double(), s["w"].detach().double(), s["offsets"].tolist()
    y = x.new_zeros(case["rows"], case["n"])
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    d = s["grad"].double() if op == "grouped_train" else None
    for e in range(case["experts"]):
        r = slice(ends[e], ends[e + 1])
        y[r] = x[r] @ w[e]
        if d is not None:
            dx[r], dw[e] = d[r] @ w[e].T, x[r].T @ d[r]
    return {"y": y} if d is None else {"y": y, "grad_x": dx, "grad_w": dw}
