"""The row, expert and grouped operators where offsets pass 2^31 elements, and side by side
on two streams and in captured graphs."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


def _skb():
    import sinkhorn_b200
    return sinkhorn_b200


def _need(gb):
    free, _ = torch.cuda.mem_get_info()
    if free < gb * 1e9:
        pytest.skip(f"needs {gb} GB of device memory")


def test_logits_beyond_2_31_elements():
    _need(16)
    skb = _skb()
    T, V = 36000, 65536
    x = torch.empty(T, V, device="cuda", dtype=torch.bfloat16)
    torch.manual_seed(0)
    for i in range(0, T, 4000):
        x[i:i + 4000].normal_()
    t = torch.arange(T, device="cuda") * 13 % V
    x.requires_grad_()
    r = skb.token_logprobs(x, t, 3)
    d, = torch.autograd.grad(r.logprob, x, torch.ones(T, device="cuda"))
    at = torch.tensor([0, 1, 32767, 32768, 32769, T - 1]).cuda()
    z = x.detach()[at].double()
    lp = torch.log_softmax(z, 1)
    want = lp.gather(1, t[at][:, None])[:, 0]
    # a lane sums 256 terms of up to (2 * 12 + 4) u each
    assert (r.logprob.detach()[at] - want).abs().max() < 400 * U32 * 12
    order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :3]
    assert torch.equal(r.top_index[at], order)
    g = -lp.exp()
    g.scatter_add_(1, t[at][:, None], torch.ones(6, 1, device="cuda", dtype=torch.float64))
    assert ((d[at].double() - g).abs() <= 2.0 ** -8 * g.abs() + 500 * U32 * lp.exp()).all()


def test_short_rows_beyond_2_31_elements():
    _need(24)
    skb = _skb()
    N, E, k = 35_000_000, 64, 2
    C = torch.empty(1, N, E, device="cuda", dtype=torch.bfloat16)
    torch.manual_seed(3)
    for i in range(0, N, 5_000_000):
        C[0, i:i + 5_000_000].normal_()
    g = torch.randn(1, E, device="cuda")
    C.requires_grad_()
    r = skb.row_logprobs(C, g, 0.5, top_k=k)
    d, = torch.autograd.grad(r.entropy, C, torch.ones(1, N, device="cuda"))
    at = torch.tensor([0, 1, 2 ** 25 - 1, 2 ** 25, 2 ** 25 + 1, N - 1]).cuda()
    x = (g[0] - C.detach()[0, at].float()).double()
    lp = torch.log_softmax(2 * x, 1)
    p = lp.exp()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(r.top_index[0, at], order)
    # |z| is below 2 * 12: (2 * 24 + 4) u a term, 8 terms a lane and 3 joins
    bound = 100 * U32 * 24
    assert (r.top_logprob.detach()[0, at] - lp.gather(1, order)).abs().max() < bound
    h = -(p * lp).sum(1)
    assert (r.entropy.detach()[0, at] - h).abs().max() < bound
    want = 2 * p * (lp + h[:, None])
    assert ((d[0, at].double() - want).abs() <= 2.0 ** -8 * want.abs() + 4 * bound * p).all()


def test_rows_beyond_2_31_elements():
    _need(22)
    skb = _skb()
    T, k, D = 270000, 4, 2048
    index = (torch.arange(T * k, device="cuda").view(T, k) * 7 + torch.arange(T, device="cuda")[:, None]) % 16
    d = skb.expert_dispatch(index, 16)
    x = torch.arange(T, device="cuda").remainder(251).to(torch.bfloat16)[:, None].expand(T, D)
    rows = skb.dispatch_rows(x, d)
    token = torch.div(d.order, k, rounding_mode="floor").long()
    assert torch.equal(rows[:, 0], x[token, 0]) and torch.equal(rows[:, -1], x[token, 0])
    out = skb.combine_rows(rows, d)
    # four times a whole number up to 250 is exact in bf16 up to its rounding
    want = (4.0 * x[:, 0].float()).to(torch.bfloat16)
    assert torch.equal(out[:, 0], want) and torch.equal(out[:, -1], want)


def test_products_beyond_2_31_elements():
    _need(16)
    skb = _skb()
    S, K, N = 540000, 4096, 64
    x = torch.empty(S, K, device="cuda", dtype=torch.bfloat16)
    torch.manual_seed(1)
    for i in range(0, S, 60000):
        x[i:i + 60000].normal_()
    w = (torch.randn(3, K, N, device="cuda") / 64).bfloat16()
    ends = [0, 100, 530000, S]
    y = skb.grouped_matmul(x, w, torch.tensor(ends, device="cuda"))
    for r, e in ((0, 0), (99, 0), (100, 1), (529999, 1), (530000, 2), (S - 1, 2)):
        want = x[r].double() @ w[e].double()
        size = x[r].double().abs() @ w[e].double().abs()
        assert ((y[r].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2 * K * U32 * size).all()
    g = torch.zeros(S, N, device="cuda", dtype=torch.bfloat16)
    g[S - 5:] = 1.0
    W = w.clone().requires_grad_()
    dw, = torch.autograd.grad(skb.grouped_matmul(x, W, torch.tensor(ends, device="cuda")), W, g)
    want = x[S - 5:].double().sum(0)
    assert (dw[:2] == 0).all()
    assert ((dw[2].double() - want[:, None]).abs() <= 2.0 ** -8 * want.abs()[:, None] + 1e-5).all()


def _work(skb, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    C, g = r(4, 1500, 700), r(4, 700)
    x, w = r(3000, 256).bfloat16(), (r(16, 256, 384) / 16).bfloat16()
    index = torch.randint(0, 16, (3000, 2), device="cuda", generator=gen)
    leaves = [t.requires_grad_() for t in (C, g, x, w)]

    def step():
        a = skb.row_logprobs(leaves[0], leaves[1], 0.2, top_k=4)
        d = skb.expert_dispatch(index, 16)
        y = skb.grouped_matmul(skb.dispatch_rows(leaves[2], d), leaves[3], d.offsets)
        o = skb.combine_rows(y, d)
        l = skb.token_logprobs(o, top_k=3)
        grads = torch.autograd.grad([a.top_logprob.sum(), a.entropy.sum(), l.entropy.sum()], leaves)
        return [v.detach() for v in (a.lse, a.top_index, o, l.top_index, *grads)]
    return step


def test_two_streams_at_once():
    skb = _skb()
    steps = [_work(skb, s) for s in (1, 2)]
    torch.cuda.synchronize()
    alone = [s() for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(5):
        got = []
        for st, step in zip(streams, steps):
            with torch.cuda.stream(st):
                got.append(step())
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_two_captured_graphs_share_nothing():
    skb = _skb()
    want = []
    for s in (3, 4):
        want.append(_work(skb, s)())
    graphs, outs, keep = [], [], []
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for s in (3, 4):
        with torch.cuda.stream(side):
            step = _work(skb, s)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(step())
        graphs.append(g)
        keep.append(step)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, st in zip(graphs, (torch.cuda.Stream(), torch.cuda.Stream())):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, outs):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_a_chain_of_dependent_launches_gives_the_same_every_time():
    # sort, copy, two products and sum start beside the end of the kernel before; two inputs
    # in turn in one buffer, so that work on stale rows shows
    skb = _skb()
    gen = torch.Generator("cuda").manual_seed(5)
    T, k, D, E = 3001, 2, 256, 16
    xs = [torch.randn(T, D, device="cuda", generator=gen).bfloat16() for _ in range(2)]
    ids = [torch.randint(0, E, (T, k), device="cuda", generator=gen) for _ in range(2)]
    w1 = torch.randn(E, D, 264, device="cuda", generator=gen).bfloat16() / 16
    w2 = torch.randn(E, 264, D, device="cuda", generator=gen).bfloat16() / 16
    gates = torch.rand(T, k, device="cuda", generator=gen)

    def chain(x, index):
        d = skb.expert_dispatch(index, E)
        y = skb.grouped_matmul(skb.dispatch_rows(x, d), w1, d.offsets)
        return skb.combine_rows(skb.grouped_matmul(y, w2, d.offsets), d, gates)

    want = []
    for i in range(2):
        want.append(chain(xs[i], ids[i]))
        torch.cuda.synchronize()
    x, index = xs[0].clone(), ids[0].clone()
    bad = torch.zeros((), device="cuda")
    for n in range(200):
        x.copy_(xs[n % 2])
        index.copy_(ids[n % 2])
        bad += (chain(x, index) != want[n % 2]).any()
    assert bad.item() == 0


def test_two_threads_with_rows_of_different_lengths():
    """A call keeps its shared memory whatever another thread launches meanwhile (the entry
    points themselves: between two calls of the wrappers the threads seldom meet)."""
    import threading
    from sinkhorn_b200 import _lib
    skb, L = _skb(), _lib.load()
    codes, begin = [], threading.Barrier(4)

    def prepared(M, top_k, N):
        C = torch.randn(2, N, M, device="cuda")
        g = torch.randn(2, M, device="cuda")
        want = skb.row_logprobs(C, g, 0.5, top_k=top_k)
        lse, ent = torch.empty(2, N, device="cuda"), torch.empty(2, N, device="cuda")
        lp = torch.empty(2, N, max(top_k, 1), device="cuda")
        idx = torch.empty(2, N, max(top_k, 1), device="cuda", dtype=torch.int64)
        stream = torch.cuda.Stream()
        args = (C.data_ptr(), 0, 2, N, M, N * M, M, 1, g.data_ptr(), 0.5, 1, None, None, None,
                top_k, lse.data_ptr(), None, ent.data_ptr(), lp.data_ptr() if top_k else None,
                idx.data_ptr() if top_k else None, None, None, 0, stream.cuda_stream)
        return args, lse, want, (C, g, ent, lp, idx, stream)

    # rows that take a CTA each, and rows that are streamed
    work = [prepared(M, k, N) for M, k, N in ((16384, 0, 5), (5000, 0, 5), (16384, 2, 300),
                                              (4100, 2, 300))]
    torch.cuda.synchronize()

    def run(args):
        begin.wait()
        codes.append({L.sk_row_logprobs(*args) for _ in range(4000)})

    threads = [threading.Thread(target=run, args=(w[0],)) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert codes == [{0}] * 4
    for _, lse, want, _ in work:
        assert torch.equal(lse, want.lse)
