"""Expert dispatch: the stable sort, rows into expert order and back, gradients."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _skb():
    import sinkhorn_b200
    return sinkhorn_b200


def plan(index, E):
    """order, position, offsets by definition."""
    flat = index.reshape(-1).tolist()
    order, offsets = [], [0]
    for e in range(E):
        order += [s for s, v in enumerate(flat) if v == e]
        offsets.append(len(order))
    position = [-1] * len(flat)
    for p, s in enumerate(order):
        position[s] = p
    order += [-1] * (len(flat) - len(order))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    return i32(order), i32(position).view(index.shape), i32(offsets)


def choices(T, k, E, seed, bad=True):
    gen = torch.Generator().manual_seed(seed)
    index = torch.randint(0, E, (T, k), generator=gen)
    if bad:
        drop = torch.rand(T, k, generator=gen) < 0.1
        index[drop] = torch.tensor([-1, E, -2 ** 40, 2 ** 40])[
            torch.randint(0, 4, (int(drop.sum()),), generator=gen)]
    return index


@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (3, 2, 5), (100, 2, 64), (700, 3, 2), (1024, 2, 31),
                                   (1025, 2, 33), (2048, 1, 257), (5000, 4, 1024), (9001, 1, 1),
                                   (4099, 5, 300)])
def test_sort(T, k, E):
    index = choices(T, k, E, T + E, bad=T > 1)
    d = _skb().expert_dispatch(index.cuda(), E)
    for got, want in zip((d.order, d.position, d.offsets), plan(index, E)):
        assert got.dtype == torch.int32 and torch.equal(got.cpu(), want)
    assert d.n_experts == E


def test_sort_of_nothing_and_of_dropped_only():
    d = _skb().expert_dispatch(torch.empty(0, 2, dtype=torch.int64).cuda(), 4)
    assert d.offsets.tolist() == [0] * 5 and d.order.numel() == 0
    d = _skb().expert_dispatch(torch.full((5000, 2), -1).cuda(), 4)
    assert d.offsets.tolist() == [0] * 5 and (d.order == -1).all() and (d.position == -1).all()


def test_sort_takes_any_integer_type_and_strides():
    index = choices(300, 4, 9, 1, bad=False)
    want = plan(index[:, ::2], 9)[0]
    for dt in (torch.int32, torch.int16, torch.uint8, torch.int64):
        d = _skb().expert_dispatch(index.to(dt).cuda()[:, ::2], 9)
        assert torch.equal(d.order.cpu(), want)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T,k,E,D", [(1, 1, 1, 1), (5, 2, 3, 7), (100, 2, 64, 2048),
                                     (33, 4, 6, 130), (257, 1, 9, 1000), (64, 3, 8, 4100)])
def test_rows_and_back(T, k, E, D, dtype):
    skb, dt = _skb(), TYPES[dtype]
    gen = torch.Generator().manual_seed(D)
    index = choices(T, k, E, D, bad=T > 1)
    order, position, offsets = plan(index, E)
    d = skb.expert_dispatch(index.cuda(), E)
    x = torch.randn(T, D, generator=gen).to(dt)
    X = x.cuda().requires_grad_()
    rows = skb.dispatch_rows(X, d)
    want = torch.where(order[:, None] >= 0, x[(order.long().clamp(min=0)) // k], torch.zeros(1, dtype=dt))
    assert torch.equal(rows.detach().cpu(), want)

    up = torch.randn(T * k, D, generator=gen).to(dt)
    dx, = torch.autograd.grad(rows, X, up.cuda())
    held = torch.where(position[..., None] >= 0, up.double()[position.long().clamp(min=0)], 0.0)
    half, tiny = torch.finfo(dt).eps / 2, torch.finfo(dt).tiny
    wx = held.sum(1)
    assert ((dx.cpu().double() - wx).abs()
            <= half * wx.abs() + k * U32 * held.abs().sum(1) + tiny).all()

    y = torch.randn(T * k, D, generator=gen).to(dt)
    w = torch.rand(T, k, generator=gen)
    Y, Wt = y.cuda().requires_grad_(), w.cuda().requires_grad_()
    out = skb.combine_rows(Y, d, Wt)
    g = torch.randn(T, D, generator=gen).to(dt)
    dy, dw = torch.autograd.grad(out, (Y, Wt), g.cuda())
    held = torch.where(position[..., None] >= 0, y.double()[position.long().clamp(min=0)], 0.0)
    terms = w.double()[..., None] * held
    wo = terms.sum(1)
    assert ((out.detach().cpu().double() - wo).abs()
            <= half * wo.abs() + k * U32 * terms.abs().sum(1) + tiny).all()
    wdy = torch.zeros(T * k, D, dtype=torch.float64)
    ok = position.reshape(-1) >= 0
    wdy[position.reshape(-1)[ok].long()] = (w.double()[..., None] * g.double()[:, None]
                                            ).reshape(T * k, D)[ok]
    # w g is rounded to fp32, then to the rows' type
    assert ((dy.cpu().double() - wdy).abs() <= (half + U32) * wdy.abs() + tiny).all()
    prod = g.double()[:, None] * held
    wdw = prod.sum(-1)
    assert dw.dtype == torch.float32
    assert ((dw.cpu().double() - wdw).abs() <= (D / 32 + 8) * U32 * prod.abs().sum(-1)).all()


def test_garbage_in_rows_behind_the_groups_does_not_show():
    skb = _skb()
    index = torch.tensor([[0, -1], [1, 0], [-1, -1]]).cuda()
    d = skb.expert_dispatch(index, 2)
    y = torch.ones(6, 8, device="cuda")
    y[3:] = float("nan")
    y.requires_grad_()
    w = torch.ones(3, 2, device="cuda", requires_grad=True)
    out = skb.combine_rows(y, d, w)
    assert out.detach().cpu()[:, 0].tolist() == [1.0, 2.0, 0.0]
    dy, dw = torch.autograd.grad(out.sum(), (y, w))
    assert (dy[3:] == 0).all() and dw.cpu().tolist() == [[8.0, 0.0], [8.0, 8.0], [0.0, 0.0]]


def test_a_plan_with_places_out_of_range_stays_in_bounds():
    """Places that are no rows count as dropped (checked in the kernels)."""
    skb = _skb()
    d = skb.expert_dispatch(torch.tensor([[0], [1], [0]]).cuda(), 2)
    d.position[1, 0] = 1000000
    x = torch.randn(3, 16, device="cuda")
    rows = skb.dispatch_rows(x, d)
    assert torch.equal(rows[0], x[0]) and torch.equal(rows[1], x[2])
    out = skb.combine_rows(torch.ones(3, 16, device="cuda"), d)
    assert out[:, 0].tolist() == [1.0, 0.0, 1.0]


@pytest.mark.parametrize("layout", ["sliced", "offset", "transposed", "expanded"])
def test_strided_rows(layout):
    skb = _skb()
    base = torch.randn(24, 40, device="cuda")
    x = {"sliced": lambda: base[::2, :24], "offset": lambda: base[:, 1:18],
         "transposed": lambda: base.t(), "expanded": lambda: base[:1].expand(10, 40)}[layout]()
    T = x.shape[0]
    d = skb.expert_dispatch(torch.arange(T).flip(0)[:, None].cuda() % 5, 5)
    rows = skb.dispatch_rows(x, d)
    assert torch.equal(rows, x[d.order.long()])
    assert torch.equal(skb.combine_rows(rows, d), x)
    up = torch.randn(T, 2 * x.shape[1], device="cuda")[:, ::2]
    X = x.detach().requires_grad_()
    g, = torch.autograd.grad(skb.combine_rows(skb.dispatch_rows(X, d), d), X, up)
    assert torch.equal(g, up)


def test_no_tokens_and_weights_of_another_type():
    skb = _skb()
    d = skb.expert_dispatch(torch.empty(0, 2, dtype=torch.int64).cuda(), 3)
    x = torch.empty(0, 5, device="cuda", requires_grad=True)
    rows = skb.dispatch_rows(x, d)
    assert rows.shape == (0, 5) and skb.combine_rows(rows, d).shape == (0, 5)
    d = skb.expert_dispatch(torch.zeros(4, 1, dtype=torch.int64).cuda(), 1)
    y = torch.ones(4, 8, device="cuda")
    w = torch.full((4, 1), 0.5, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = skb.combine_rows(y, d, w)
    dw, = torch.autograd.grad(out.sum(), w)
    assert (out == 0.5).all() and dw.dtype == torch.bfloat16 and (dw == 8).all()


def test_captured_and_replayed_on_another_stream():
    skb = _skb()
    index = choices(3000, 2, 16, 3).cuda()
    x = torch.randn(3000, 64, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        skb.combine_rows(skb.dispatch_rows(x, skb.expert_dispatch(index, 16)),
                         skb.expert_dispatch(index, 16))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            d = skb.expert_dispatch(index, 16)
            out = skb.combine_rows(skb.dispatch_rows(x, d), d)
    torch.cuda.synchronize()
    index.copy_(choices(3000, 2, 16, 4))
    graph.replay()
    torch.cuda.synchronize()
    order, position, _ = plan(index.cpu(), 16)
    assert torch.equal(d.order.cpu(), order)
    assert torch.equal(out.cpu(), x.cpu() * (position >= 0).sum(1, keepdim=True))
