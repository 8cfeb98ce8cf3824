"""The operators together: a layer of experts routed by the Sinkhorn plan."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


def _skb():
    import sinkhorn_b200
    return sinkhorn_b200


def test_assign_is_the_normalised_plan():
    skb = _skb()
    gen = torch.Generator().manual_seed(0)
    C = torch.rand(2, 40, 24, generator=gen).cuda()
    mb = (torch.rand(2, 24, generator=gen) > 0.2).cuda()
    out = skb.sinkhorn(C, epsilon=0.1, mask_b=mb, max_iters=200)
    t = mb.int().argmax(1, keepdim=True).expand(2, 40).contiguous()
    r = out.assign(C, 0.1, top_k=3, targets=t, mask_b=mb)
    P = out.transport_plan(C, 0.1, mask_b=mb).double()
    p = P / P.sum(-1, keepdim=True)
    # P rounds its exponent (up to 100 for these costs) and each entry to fp32
    tol = 128 * U32
    assert (r.logprob.double() - p.gather(-1, t[..., None])[..., 0].log()).abs().max() < tol * 8
    v = p.topk(3).values
    assert (r.top_logprob.double().exp() - v).abs().max() < tol * 8
    h = -(p * torch.where(p > 0, p, torch.ones_like(p)).log()).sum(-1)
    assert (r.entropy.double() - h).abs().max() < tol * 16


def test_routing_balances_the_experts():
    skb = _skb()
    gen = torch.Generator().manual_seed(1)
    scores = (torch.randn(4096, 16, generator=gen) + 2 * torch.randn(16, generator=gen)).cuda()
    r = skb.sinkhorn_route(scores, 1, epsilon=0.05, max_iters=500, threshold=1e-6)
    counts = r.dispatch.offsets.diff().float()
    alone = torch.bincount(scores.argmax(1), minlength=16).float()
    # the expected loads are equal; the choices' loads come near them, the scores' do not
    assert counts.max() < 2 * 4096 / 16 < alone.max()
    assert r.index.shape == (4096, 1) and (r.gates == 1).all()


def test_masked_tokens_go_nowhere():
    skb = _skb()
    scores = torch.randn(50, 8, generator=torch.Generator().manual_seed(2)).cuda()
    mask = torch.ones(50, dtype=torch.bool).cuda()
    mask[7], mask[40:] = False, False
    s = scores.clone().requires_grad_()
    r = skb.sinkhorn_route(s, 2, mask=mask)
    assert (r.index[~mask] == -1).all() and (r.index[mask] >= 0).all()
    assert (r.gates[~mask] == 0).all() and int(r.dispatch.offsets[-1]) == 2 * int(mask.sum())
    d, = torch.autograd.grad(r.gates[:, 0].sum(), s)
    assert torch.isfinite(d).all() and (d[~mask] == 0).all()


@pytest.mark.parametrize("T,E,D,H,k,dtype", [
    (300, 4, 64, 96, 2, torch.bfloat16), (257, 8, 40, 24, 1, torch.float16),
    (64, 3, 33, 17, 3, torch.bfloat16), (1, 2, 16, 16, 1, torch.bfloat16)])
def test_layer_against_a_loop_over_the_tokens(T, E, D, H, k, dtype):
    skb = _skb()
    gen = torch.Generator().manual_seed(T)
    r = lambda *s: torch.randn(*s, generator=gen)
    x, scores = r(T, D).to(dtype), r(T, E)
    w1, w2 = (r(E, D, H) / D ** 0.5).to(dtype), (r(E, H, D) / H ** 0.5).to(dtype)
    mask = torch.ones(T, dtype=torch.bool)
    mask[T // 2:T // 2 + T // 10] = False
    leaves = [t.cuda().requires_grad_() for t in (x, scores, w1, w2)]
    out, route = skb.sinkhorn_experts(*leaves, top_k=k, epsilon=0.2, mask=mask.cuda())
    up = r(T, D).to(dtype)
    grads = torch.autograd.grad(out, leaves, up.cuda())

    # the same in 64 bits, with the routes and the column potential as they came
    index = route.index.cpu()
    ref = [t.double().requires_grad_() for t in (x, scores, w1, w2)]
    C = -scores[None].cuda()
    g = skb.sinkhorn(C, epsilon=0.2, mask_a=mask[None].cuda(), max_iters=50,
                     threshold=1e-3).g.double().cpu()
    lp = torch.log_softmax((g[0] + ref[1]) / 0.2, -1)
    p = lp.gather(1, index.clamp(min=0)).exp() * (index >= 0)
    gates = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    want = torch.zeros(T, D, dtype=torch.float64)
    for j in range(k):
        e = index[:, j].clamp(min=0)
        h = torch.nn.functional.silu(torch.einsum("td,tdh->th", ref[0], ref[2][e]))
        y = torch.einsum("th,thd->td", h, ref[3][e])
        want = want + (gates[:, j] * (index[:, j] >= 0))[:, None] * y
    wants = torch.autograd.grad(want, ref, up.double())
    # six results rounded to 16 bits lie on the longest way (product, activation, product
    # and their gradients), each off by half a step of a value of the result's size
    half = torch.finfo(dtype).eps / 2
    for got, w in zip([out] + list(grads), [want] + list(wants)):
        got, w = got.detach().double().cpu(), w.detach()
        assert torch.isfinite(got).all()
        assert (got - w).norm() <= 6 * half * w.norm() + 1e-6
    assert (grads[1].cpu()[~mask] == 0).all() and (grads[0].cpu()[~mask] == 0).all()


def test_layer_step_twice_is_the_same():
    skb = _skb()
    gen = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen).cuda()
    x, scores = r(500, 64).bfloat16().requires_grad_(), r(500, 8).requires_grad_()
    w1, w2 = (r(8, 64, 128) / 8).bfloat16().requires_grad_(), (r(8, 128, 64) / 11).bfloat16().requires_grad_()

    def step():
        out, _ = skb.sinkhorn_experts(x, scores, w1, w2, top_k=2)
        lp = skb.token_logprobs(out, torch.arange(500).cuda() % 64)
        return torch.autograd.grad(lp.logprob.sum(), (x, scores, w1, w2))

    for a, b in zip(step(), step()):
        assert torch.equal(a, b) and torch.isfinite(a).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_padding_tokens_hold_reaches_nothing(bad):
    skb = _skb()
    gen = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=gen)
    scores, x = r(60, 8), r(60, 32).bfloat16()
    w1, w2 = (r(8, 32, 48) / 6).bfloat16(), (r(8, 48, 32) / 7).bfloat16()
    mask = torch.ones(60, dtype=torch.bool)
    mask[11], mask[50:] = False, False
    got = []
    for fill in (0.0, bad):
        s, y = scores.clone(), x.clone()
        s[~mask], y[~mask] = fill, fill
        leaves = [v.cuda().requires_grad_() for v in (y, s, w1, w2)]
        out, route = skb.sinkhorn_experts(*leaves, top_k=2, epsilon=0.2, mask=mask.cuda())
        got.append([out.detach(), route.gates.detach(), route.index,
                    *torch.autograd.grad(out.float().square().sum() + route.rows.entropy.sum(),
                                         leaves)])
    for a, b in zip(*got):
        assert torch.equal(a, b) and torch.isfinite(b).all()
    assert all((v[~mask.cuda()] == 0).all() for v in (got[1][0], got[1][3], got[1][4]))


def test_a_nan_score_shows_in_its_own_token():
    skb = _skb()
    gen = torch.Generator().manual_seed(9)
    r = lambda *s: torch.randn(*s, generator=gen).cuda()
    scores, x = r(40, 8), r(40, 16).bfloat16()
    w1, w2 = r(8, 16, 16).bfloat16(), r(8, 16, 16).bfloat16()
    scores[3, 2] = float("nan")
    scores[7] = float("nan")
    s = scores.requires_grad_()
    out, route = skb.sinkhorn_experts(x, s, w1, w2, top_k=2)
    d, = torch.autograd.grad(out.float().sum(), s)
    others = torch.ones(40, dtype=torch.bool)
    others[3] = others[7] = False
    assert out[3].isnan().all() and route.gates[3].isnan().all() and d[3].isnan().any()
    assert (route.index[7] == -1).all() and route.rows.lse[0, 7].isnan() and (out[7] == 0).all()
    assert torch.isfinite(out[others]).all() and torch.isfinite(d[others]).all()
