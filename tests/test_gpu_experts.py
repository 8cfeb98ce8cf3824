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


def held_by(d):
    """place -> slot of a plan: slot s holds place p where position[s] = p, order[p] = s and p
    lies before the last offset."""
    order, position = d.order.tolist(), d.position.reshape(-1).tolist()
    n = min(len(order), int(d.offsets[-1]))
    return {p: s for s, p in enumerate(position) if 0 <= p < n and order[p] == s}


def _edit(d, how):
    if how == "places dropped":
        d.position[1, 0], d.position[7, 1], d.position[20, 0] = -1, -1, 10 ** 6
    elif how == "order dropped":
        d.order[3], d.order[17] = -1, 2 ** 30
    elif how == "two slots at one place":
        d.position[4, 0], d.position[9, 1] = d.position[5, 1], d.position[6, 0]
    elif how == "fewer rows":
        d.offsets[-1] -= 9
    elif how == "more rows":
        d.offsets[-1] = 10 ** 6
    elif how == "places exchanged":  # in both: a plan as good as before
        a, b = int(d.position[2, 0]), int(d.position[12, 1])
        d.position[2, 0], d.position[12, 1] = b, a
        d.order[a], d.order[b] = 12 * 2 + 1, 2 * 2


@pytest.mark.parametrize("how", ["places dropped", "order dropped", "two slots at one place",
                                 "fewer rows", "more rows", "places exchanged"])
@pytest.mark.parametrize("dtype,D", [("fp32", 64), ("fp32", 130), ("fp32", 33), ("bf16", 1000),
                                     ("bf16", 36), ("fp16", 34), ("fp16", 77)])
def test_places_that_no_slot_holds_are_zero(how, dtype, D):
    """Plans that a caller has edited, as for experts over their capacity: nothing that the
    memory held before shows."""
    skb, dt = _skb(), TYPES[dtype]
    T, k, E = 40, 2, 5
    gen = torch.Generator().manual_seed(D)
    d = skb.expert_dispatch(torch.randint(0, E, (T, k), generator=gen).cuda(), E)
    _edit(d, how)
    held = held_by(d)
    x = torch.randn(T, D, generator=gen).to(dt)
    y = torch.randn(T * k, D, generator=gen).to(dt)
    w, up = torch.rand(T, k, generator=gen), torch.randn(T, D, generator=gen).to(dt)

    def stale():  # what torch.empty gives next
        keep = [torch.full((T * k, D), float("nan"), device="cuda", dtype=dt) for _ in range(4)]
        del keep

    stale()
    rows = skb.dispatch_rows(x.cuda(), d)
    want = torch.zeros(T * k, D, dtype=dt)
    for p, s in held.items():
        want[p] = x[s // k]
    assert torch.equal(rows.cpu(), want)

    Y, W = y.cuda().requires_grad_(), w.cuda().requires_grad_()
    out = skb.combine_rows(Y, d, W)
    stale()
    dy, dw = torch.autograd.grad(out, (Y, W), up.cuda())
    wout, wdy = torch.zeros(T, D, dtype=torch.float64), torch.zeros(T * k, D, dtype=torch.float64)
    wdw, size = torch.zeros(T * k, dtype=torch.float64), torch.zeros(T * k, dtype=torch.float64)
    terms = torch.zeros(T, D, dtype=torch.float64)
    for p, s in held.items():
        a = w.reshape(-1)[s].double()
        wout[s // k] += a * y[p].double()
        terms[s // k] += (a * y[p].double()).abs()
        wdy[p] = a * up[s // k].double()
        wdw[s] = (up[s // k].double() * y[p].double()).sum()
        size[s] = (up[s // k].double() * y[p].double()).abs().sum()
    half, tiny = torch.finfo(dt).eps / 2, torch.finfo(dt).tiny
    assert ((out.detach().double().cpu() - wout).abs() <= half * wout.abs() + k * U32 * terms
            + tiny).all()
    assert ((dy.double().cpu() - wdy).abs() <= (half + U32) * wdy.abs() + tiny).all()
    # a lane adds up to D / 32 products, the warp five sums
    assert ((dw.double().cpu().reshape(-1) - wdw).abs() <= (D / 32 + 8) * U32 * size).all()
    # the gradient of dispatch_rows is combine_rows of the same plan
    X = x.cuda().requires_grad_()
    dx, = torch.autograd.grad(skb.dispatch_rows(X, d), X, y.cuda())
    assert torch.equal(dx, skb.combine_rows(y.cuda(), d))


def test_products_of_a_plan_with_dropped_places():
    skb = _skb()
    gen = torch.Generator().manual_seed(1)
    d = skb.expert_dispatch(torch.randint(0, 3, (50, 2), generator=gen).cuda(), 3)
    d.position[10:20] = -1
    x = torch.randn(50, 64, generator=gen).bfloat16().cuda().requires_grad_()
    w = (torch.randn(3, 64, 48, generator=gen) / 8).bfloat16().cuda().requires_grad_()
    junk = [torch.full((100, n), float("nan"), device="cuda", dtype=torch.bfloat16)
            for n in (64, 48) * 3]
    del junk
    out = skb.combine_rows(skb.grouped_matmul(skb.dispatch_rows(x, d), w, d.offsets), d)
    dx, dw = torch.autograd.grad(out.float().sum(), (x, w))
    for v in (out, dx):
        assert torch.isfinite(v).all() and (v[10:20] == 0).all() and (v[:10] != 0).any()
    for e in range(3):  # every row of dW_e's columns is the sum of the expert's held rows
        held = [s // 2 for s in d.order[int(d.offsets[e]):int(d.offsets[e + 1])].tolist()
                if not 10 <= s // 2 < 20]
        rows = x.detach().cpu()[held].double()
        # the sum of n values, in fp32, rounded once
        bound = 2.0 ** -8 * rows.sum(0).abs() + 2 * len(held) * U32 * rows.abs().sum(0)
        assert ((dw[e].double().cpu() - rows.sum(0)[:, None]).abs() <= bound[:, None]).all()


def test_entry_points_without_the_order_agree_on_plans_of_the_sort():
    from sinkhorn_b200 import _lib
    skb, L = _skb(), _lib.load()
    T, k, E, D = 60, 2, 5, 72
    d = skb.expert_dispatch(choices(T, k, E, 8).cuda(), E)
    x, w = torch.randn(T, D, device="cuda"), torch.rand(T, k, device="cuda")
    y = torch.randn(T * k, D, device="cuda").requires_grad_()
    out = skb.combine_rows(y, d, w.requires_grad_())
    dy, dw = torch.autograd.grad(out, (y, w), x)
    new = lambda *s: torch.full(s, float("nan"), device="cuda")
    rows, sums, gy, gw = new(T * k, D), new(T, D), new(T * k, D), new(T, k)
    s, p = torch.cuda.current_stream().cuda_stream, (d.position.data_ptr(), d.offsets.data_ptr())
    ptr = lambda t: t.data_ptr()
    assert L.sk_dispatch_rows(ptr(x), 0, T, k, D, D, *p, E, ptr(rows), s) == 0
    assert L.sk_combine_rows(ptr(y), 0, T, k, D, D, *p, E, ptr(w), ptr(sums), s) == 0
    assert L.sk_combine_rows_backward(ptr(x), ptr(y), 0, T, k, D, D, D, *p, E, ptr(w), ptr(gy),
                                      ptr(gw), s) == 0
    assert torch.equal(rows, skb.dispatch_rows(x, d)) and torch.equal(sums, out)
    assert torch.equal(gy, dy) and torch.equal(gw, dw)


@pytest.mark.parametrize("T,k,E", [(606209, 1, 300), (700001, 1, 1024), (1500007, 4, 256),
                                   (5000001, 1, 1), (2600000, 3, 7)])
def test_sort_of_many_slots(T, k, E):
    """More slots than one run of 2048 to a CTA."""
    gen = torch.Generator("cuda").manual_seed(T)
    index = torch.randint(-1, E + 1, (T, k), device="cuda", generator=gen)
    d = _skb().expert_dispatch(index, E)
    flat = index.reshape(-1)
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.sort(key, stable=True).indices
    counts = torch.bincount(key, minlength=E + 1)
    held = int(counts[:E].sum())
    offsets = torch.cat([counts.new_zeros(1), counts[:E].cumsum(0)])
    position = torch.full_like(flat, -1)
    position[order[:held]] = torch.arange(held, device="cuda")
    assert torch.equal(d.offsets, offsets.int())
    assert torch.equal(d.order[:held], order[:held].int()) and (d.order[held:] == -1).all()
    assert torch.equal(d.position.reshape(-1), position.int())
