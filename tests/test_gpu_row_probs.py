"""Row and token log probabilities (row_logprobs, token_logprobs) against a plain
64-bit implementation, at the sizes, layouts and masks where they can go wrong.

Tolerances count roundings of fp32 (u = 2^-24). A term 2^y has relative error
(2 |z| + 4) u: the difference x - m, the scale and the product each round once
(|z| u apiece at most), ex2.approx is good to two units of the last place. A sum of n such
terms adds (chain + 8) u with `chain` the longest run of additions in one lane.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _skb():
    import sinkhorn_b200
    return sinkhorn_b200


def plain(x, scale, targets=None, k=0):
    """x (rows, M) fp64 on the CPU with -inf where masked: the outputs by definition."""
    z = x * scale
    M = x.shape[1]
    lse = torch.logsumexp(z, 1)
    none = lse == -math.inf
    lp = torch.where(none[:, None], torch.full_like(z, -math.inf), z - lse[:, None])
    p = lp.exp()
    ent = -(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum(1)
    out = {"lse": lse, "entropy": torch.where(none, torch.zeros_like(ent), ent), "lp": lp, "p": p}
    if targets is not None:
        t = targets.clamp(0, M - 1)
        got = lp.gather(1, t[:, None])[:, 0]
        got = torch.where(targets < 0, torch.zeros_like(got), got)
        out["logprob"] = torch.where(targets >= M, torch.full_like(got, math.nan), got)
    if k:
        idx = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :k]
        held = x.gather(1, idx) > -math.inf
        out["top_index"] = torch.where(held, idx, -1)
        out["top_logprob"] = torch.where(held, lp.gather(1, idx), -math.inf)
    return out


def _bounds(ref, M):
    """Absolute bounds of lse / log p and of the entropy for each row."""
    lp = ref["lp"].clamp(min=-110.0)
    far = lp.max(1).values[:, None] - lp  # |z| of each term
    w = ref["p"]
    chain = (M / 32 if M <= 8192 else M / 256) + 40
    rel = (w * (2 * far + 4)).sum(1) * U32 + (chain + 8) * U32  # of the sum
    ent = rel * (1 + ref["entropy"]) + (w * far * (2 * far + 6)).sum(1) * U32 + 8 * U32
    return rel, ent


def close(got, want, bound):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got))
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    assert torch.equal(got.isnan(), want.isnan())
    over = ((got - want).abs() - bound)[fine]
    assert not (over > 0).any(), float(over.max())


def check(r, ref, M, k=0):
    rel, ent = _bounds(ref, M)
    rows = ref["lse"].shape[0]
    size = lambda t: (3 * torch.where(torch.isfinite(t), t, 0.0).abs() + 8) * U32
    close(r.lse.reshape(rows), ref["lse"], rel + size(ref["lse"]))
    close(r.entropy.reshape(rows), ref["entropy"], ent)
    if "logprob" in ref:
        close(r.logprob.reshape(rows), ref["logprob"], rel + size(ref["logprob"]))
    if k:
        assert r.top_index.dtype == torch.int64
        assert torch.equal(r.top_index.reshape(rows, k).cpu(), ref["top_index"])
        close(r.top_logprob.reshape(rows, k), ref["top_logprob"],
              rel[:, None] + size(ref["top_logprob"]))


def make(B, N, M, dtype, seed, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    C = (spread * torch.randn(B, N, M, generator=gen)).to(dtype)
    g = 0.5 * torch.randn(B, M, generator=gen)
    t = torch.randint(0, M, (B, N), generator=gen)
    ma = torch.rand(B, N, generator=gen) > 0.2
    mb = torch.rand(B, M, generator=gen) > 0.2
    return C, g, t, ma, mb


def shaped(C, g, ma=None, mb=None):
    """x of the cost form, in fp32 as the operator orders it, widened."""
    x = (-C.float() if g is None else g[:, None] - C.float())
    if mb is not None:
        x = x.masked_fill(~mb[:, None], -math.inf)
    if ma is not None:
        x = x.masked_fill(~ma[..., None], -math.inf)
    return x.double().reshape(-1, C.shape[-1])


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,N,M,k", [
    (1, 1, 1, 1), (2, 3, 2, 2), (1, 5, 7, 3), (3, 17, 33, 5), (2, 9, 64, 2), (1, 33, 128, 8),
    (2, 5, 255, 32), (1, 4, 513, 1), (1, 3, 1027, 20), (1, 2, 4099, 7), (2, 2, 16387, 32),
    (1, 1, 70001, 20), (1, 2500, 1536, 3), (1, 2500, 4091, 3),
])
def test_rows_of_a_cost(B, N, M, k, dtype):
    C, g, t, ma, mb = make(B, N, M, TYPES[dtype], 1000 * M + k)
    t[..., 0] = -7 if M > 1 else t[..., 0]
    eps = 0.25
    r = _skb().row_logprobs(C.cuda(), g.cuda(), eps, t.cuda(), k, ma.cuda(), mb.cuda())
    check(r, plain(shaped(C, g, ma, mb), 1 / eps, t.reshape(-1), k), M, k)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T,V,k", [(1, 131072, 20), (3, 50001, 5), (700, 9001, 0), (1, 3, 0),
                                   (40, 2047, 32), (300, 96, 4)])
def test_tokens_of_logits(T, V, k, dtype):
    logits = (3 * torch.randn(T, V, generator=torch.Generator().manual_seed(V))).to(TYPES[dtype])
    t = torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(1))
    r = _skb().token_logprobs(logits.cuda(), t.cuda(), k, temperature=0.7)
    check(r, plain(logits.double(), 1 / 0.7, t, k), V, k)
    assert (r.top_index is None) == (k == 0)


def test_no_potential_no_mask_and_no_target():
    C, _, _, _, _ = make(2, 6, 100, torch.float32, 3)
    r = _skb().row_logprobs(C.cuda(), epsilon=1.0)
    check(r, plain(shaped(C, None), 1.0), 100)
    assert r.logprob is None and r.top_logprob is None


@pytest.mark.parametrize("layout", ["sliced", "transposed", "broadcast", "offset", "column"])
def test_layouts(layout):
    gen = torch.Generator().manual_seed(5)
    base = torch.randn(3, 40, 70, generator=gen).cuda()
    C = {"sliced": lambda: base[:, 3:29, 5:66], "transposed": lambda: base.transpose(1, 2),
         "broadcast": lambda: base[:1].expand(3, 40, 70), "offset": lambda: base[:, :, 1:],
         "column": lambda: base[:, :, 9:10]}[layout]()
    k = min(4, C.shape[2])
    r = _skb().row_logprobs(C, None, 0.5, top_k=k)
    check(r, plain(shaped(C.cpu(), None), 2.0, k=k), C.shape[2], k)
    X = C.detach().requires_grad_()
    r = _skb().row_logprobs(X, None, 0.5, top_k=k)
    d, = torch.autograd.grad(r.top_logprob.sum() + r.entropy.sum(), X)
    Y = C.detach().cpu().double().requires_grad_()
    lp = torch.log_softmax(-2 * Y, -1)
    want, = torch.autograd.grad(lp.topk(k).values.sum() - (lp.exp() * lp).sum(), Y)
    assert d.shape == C.shape
    # |dz| is below k + |log p| p + ...: 64 roundings of values up to 2 (k + 4)
    assert (d.cpu().double() - want).abs().max() < 64 * U32 * 2 * (k + 4)


def test_ties_go_to_the_lowest_column():
    X = torch.zeros(5, 3000)
    X[1, 2000:2040] = 1.0
    X[2, ::7] = 2.0
    X[3] = -0.0
    X[3, 5::2] = 0.0
    X[4] = torch.arange(3000) // 100
    for V in (3000, 61):
        x = X[:, :V].contiguous()
        r = _skb().token_logprobs(x.cuda(), top_k=32)
        check(r, plain(x.double(), 1.0, k=32), V, 32)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,N,M,k", [(1, 5001, 2, 2), (70, 1, 8, 8), (3, 333, 31, 1),
                                     (2, 2500, 63, 7), (1, 40, 64, 0), (1, 6, 64, 8),
                                     (1, 1700, 65, 8), (2, 31, 100, 3), (2, 33, 127, 8),
                                     (1, 21000, 128, 2), (1, 65, 129, 8), (1, 65, 128, 9),
                                     (2, 1111, 200, 6), (1, 40, 256, 8), (3, 33, 257, 2),
                                     (1, 700, 511, 1), (2, 10, 512, 2), (1, 9, 512, 3)])
def test_short_rows(B, N, M, k, dtype):
    # rows that start anywhere, with a potential and masks, and as they are
    C, g, t, ma, mb = make(B, N, M + 3, TYPES[dtype], 100 * M + k, spread=3.0)
    C = C[..., 2:2 + M] if N % 2 else C[..., :M].contiguous()
    g, mb, t = g[:, :M], mb[:, :M], t.clamp(max=M - 1)
    on = C.cuda() if N % 2 == 0 else torch.cat([C, C, C], 2).cuda()[..., M:2 * M]
    r = _skb().row_logprobs(on, g.cuda(), 0.25, t.cuda(), k, ma.cuda(), mb.cuda())
    check(r, plain(shaped(C, g, ma, mb), 4.0, t.reshape(-1), k), M, k)
    r = _skb().row_logprobs(on, g.cuda(), 0.25, t.cuda(), k)
    check(r, plain(shaped(C, g), 4.0, t.reshape(-1), k), M, k)
    r = _skb().token_logprobs(on, t.cuda(), k)
    check(r, plain(C.double().reshape(-1, M), 1.0, t.reshape(-1), k), M, k)


def test_short_rows_of_equal_values_and_of_few():
    x = torch.zeros(6, 61)
    x[1] = -0.0
    x[1, 5::2] = 0.0
    x[2] = torch.arange(61) // 10
    x[3] = -math.inf
    x[4] = -math.inf
    x[4, 60] = x[4, 3] = 1.0
    x[5, :30] = -math.inf
    r = _skb().token_logprobs(x.cuda(), top_k=8)
    check(r, plain(x.double(), 1.0, k=8), 61, 8)
    x[2, 7] = math.nan
    x[5] = math.nan
    r = _skb().token_logprobs(x.cuda(), top_k=8)
    assert r.lse[[2, 5]].isnan().all() and r.entropy[[2, 5]].isnan().all()
    assert torch.isfinite(r.lse[[0, 1, 4]]).all() and (r.lse[3] == -math.inf)
    assert (r.top_index[2] == torch.arange(60, 61).cuda()).any() and (r.top_index[2] != 7).all()
    assert (r.top_index[5] == -1).all()


@pytest.mark.parametrize("V", [100, 5000, 40000])
def test_sorted_rows(V):
    up = torch.linspace(-3, 3, V).repeat(3, 1)
    up[1] = up[1].flip(0)
    r = _skb().token_logprobs(up.cuda(), top_k=32)
    check(r, plain(up.double(), 1.0, k=32), V, 32)


@pytest.mark.parametrize("M", [5, 300, 9000])
def test_rows_without_columns_and_masked_garbage(M):
    C, g, t, ma, mb = make(2, 6, M, torch.float32, M)
    C[:, :, 0] = math.nan
    C[:, 1, 1] = -math.inf
    mb[:, :2] = False
    mb[0] = False  # the whole first item: every row empty
    ma[1, 0] = False
    C[1, 2, :] = math.inf  # a cost of +inf everywhere leaves nothing
    t[1, 3] = 0            # a masked target
    X, G = C.cuda().requires_grad_(), g.cuda().requires_grad_()
    r = _skb().row_logprobs(X, G, 0.5, t.cuda(), 4, ma.cuda(), mb.cuda())
    ref = plain(shaped(C, g, ma, mb), 2.0, t.reshape(-1), 4)
    check(r, ref, M, 4)
    assert (r.lse[0] == -math.inf).all() and (r.entropy[0] == 0).all()
    assert (r.top_index[0] == -1).all() and (r.top_logprob[0] == -math.inf).all()
    ones = [torch.ones_like(v) for v in (r.lse, r.logprob, r.entropy, r.top_logprob)]
    dC, dg = torch.autograd.grad((r.lse, r.logprob, r.entropy, r.top_logprob), (X, G), ones)
    assert torch.isfinite(dC).all() and torch.isfinite(dg).all()
    assert (dC[0] == 0).all() and (dC[1, 0] == 0).all() and (dC[1, 2] == 0).all()
    assert (dC[:, :, :2] == 0).all() and (dg[0] == 0).all()


@pytest.mark.parametrize("V", [40, 3000, 70000])
def test_nan_and_infinite_logits_show(V):
    x = torch.randn(4, V, generator=torch.Generator().manual_seed(0))
    x[1, V // 2] = math.nan
    x[2, V - 1] = math.inf
    x[3] = math.nan
    r = _skb().token_logprobs(x.cuda(), torch.zeros(4, dtype=torch.int64).cuda(), 3)
    for v in (r.lse, r.logprob, r.entropy):
        assert torch.isfinite(v[0]) and not torch.isfinite(v[1:]).any()
    assert r.lse[1].isnan() and r.lse[3].isnan() and r.entropy[2].isnan()
    assert r.top_index[2, 0] == V - 1
    assert torch.equal(r.top_index[3].cpu(), torch.full((3,), -1))


def test_target_out_of_range_is_nan_and_passes_nothing():
    x = torch.randn(3, 50, generator=torch.Generator().manual_seed(0)).cuda().requires_grad_()
    r = _skb().token_logprobs(x, torch.tensor([50, -1, 2 ** 40]).cuda())
    assert r.logprob[0].isnan() and r.logprob[1] == 0 and r.logprob[2].isnan()
    d, = torch.autograd.grad(r.logprob, x, torch.ones(3).cuda())
    assert (d == 0).all()


def test_no_rows():
    x = torch.empty(0, 7, device="cuda", requires_grad=True)
    r = _skb().token_logprobs(x, torch.empty(0, dtype=torch.int64, device="cuda"), 2)
    assert r.lse.shape == (0,) and r.top_index.shape == (0, 2)
    d, = torch.autograd.grad(r.logprob.sum() + r.lse.sum(), x)
    assert d.shape == x.shape
    C = torch.empty(2, 0, 5, device="cuda")
    g = torch.zeros(2, 5, device="cuda", requires_grad=True)
    r = _skb().row_logprobs(C, g, 0.1)
    dg, = torch.autograd.grad(r.lse.sum(), g)
    assert (dg == 0).all()


def _gradients(C, g, eps, t, k, ma, mb, ups):
    """fp64 gradients of the definition by autograd (rows that are empty left out)."""
    Y, G = C.double().requires_grad_(), g.double().requires_grad_()
    x = G[:, None] - Y
    z = torch.where(mb[:, None], x / eps, -1e9)
    lp = torch.log_softmax(z, -1)
    p = lp.exp()
    live = ma[..., None] & mb.any(1)[:, None, None]
    order = torch.sort((g[:, None] - C.float()).masked_fill(~mb[:, None], -math.inf), dim=-1,
                       descending=True, stable=True).indices[..., :k]
    given = (t >= 0) & mb.gather(1, t.clamp(min=0))
    loss = (torch.where(given[..., None] & live, lp.gather(-1, t.clamp(min=0)[..., None]), 0.0)
            [..., 0] * ups[1].double()).sum()
    loss = loss + (torch.logsumexp(z, -1) * live[..., 0] * ups[0].double()).sum()
    h = -(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum(-1)
    loss = loss + (h * live[..., 0] * ups[2].double()).sum()
    present = mb[:, None].expand(C.shape).gather(-1, order) & live
    loss = loss + (torch.where(present, lp.gather(-1, order), 0.0) * ups[3].double()).sum()
    return torch.autograd.grad(loss, (Y, G)), p.detach(), lp.detach()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,N,M,k,masked", [
    (1, 1, 1, 1, False), (2, 5, 7, 3, True), (1, 300, 64, 2, False), (3, 40, 65, 8, True),
    (2, 70, 256, 32, True), (1, 130, 1031, 4, True), (2, 3, 9001, 5, False),
])
def test_gradients(B, N, M, k, masked, dtype):
    eps = 0.5
    C, g, t, ma, mb = make(B, N, M, TYPES[dtype], M + k)
    if not masked:
        ma[:], mb[:] = True, True
    if M > 1:
        t[..., 0] = -1
    gen = torch.Generator().manual_seed(9)
    ups = [torch.randn(s, generator=gen) for s in ((B, N),) * 3 + ((B, N, k),)]
    X, G = C.cuda().requires_grad_(), g.cuda().requires_grad_()
    r = _skb().row_logprobs(X, G, eps, t.cuda(), k, ma.cuda(), mb.cuda())
    outs = (r.lse, r.logprob, r.entropy, r.top_logprob)
    dC, dg = torch.autograd.grad(outs, (X, G), [u.cuda() for u in ups])
    assert dC.dtype == C.dtype and dg.dtype == torch.float32
    (wC, wg), p, lp = _gradients(C, g, eps, t, k, ma, mb, ups)
    # p carries (2 |log p| + chain + 12) u, its factor sums k + 3 terms of size `big`
    chain = M / 32 + 48
    big = ups[0].abs() + ups[1].abs() + ups[3].abs().sum(-1) + 2 * ups[2].abs() * 16
    lpc = lp.clamp(min=-110.0).abs()
    err = (p * (2 * lpc + chain + k + 24) * (big[..., None] + ups[2].abs()[..., None] * lpc)
           + (k + 4) * big[..., None] * (p + 1e-3)) * U32 / eps
    err = err + 4 * U32 * wC.abs()
    half = torch.finfo(TYPES[dtype]).eps / 2
    tiny = torch.finfo(TYPES[dtype]).tiny
    off = (dC.double().cpu() - wC).abs()
    assert (off <= err + half * wC.abs() + tiny).all(), float((off - err).max())
    off = (dg.double().cpu() - wg).abs()
    assert (off <= err.sum(1) + (N + 8) * U32 * wC.abs().sum(1)).all()


def test_gradient_against_differences():
    C, g, t, _, _ = make(1, 3, 11, torch.float32, 2)
    C, g, t = C.cuda(), g.cuda(), t.cuda()

    def loss(C, g):
        r = _skb().row_logprobs(C, g, 0.7, t, 2)
        return (r.logprob.double().sum() + 0.3 * r.entropy.double().sum()
                + 0.2 * r.lse.double().sum() + 0.5 * r.top_logprob.double().sum())

    X, G = C.clone().requires_grad_(), g.clone().requires_grad_()
    dC, dg = torch.autograd.grad(loss(X, G), (X, G))
    h = 2.0 ** -6
    for at in [(0, 0, 0), (0, 1, 5), (0, 2, 10)]:
        e = torch.zeros_like(C)
        e[at] = h
        num = float(loss(C + e, g) - loss(C - e, g)) / (2 * h)
        # the third derivative, some tens in z / 0.7^3, times h^2 / 6; and 60 u / h of rounding
        assert abs(num - float(dC[at])) < 50 * h * h + 60 * U32 / h
    e = torch.zeros_like(g)
    e[0, 4] = h
    num = float(loss(C, g + e) - loss(C, g - e)) / (2 * h)
    assert abs(num - float(dg[0, 4])) < 150 * h * h + 60 * U32 / h


@pytest.mark.parametrize("V", [64, 5001])
def test_token_gradient_odd_rows(V):
    """Rows that start off the 16-byte grid, the gradient in the logits' type."""
    x = torch.randn(9, V, generator=torch.Generator().manual_seed(4)).bfloat16()
    t = torch.arange(9) * 7 % V
    X = x.cuda().requires_grad_()
    r = _skb().token_logprobs(X, t.cuda())
    d, = torch.autograd.grad(-r.logprob.sum(), X)
    p = torch.softmax(x.double(), 1)
    want = p.clone()
    want[torch.arange(9), t] -= 1
    assert ((d.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 300 * U32 * p).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("N,M,k", [(2500, 4091, 3), (2500, 1999, 0), (700, 9001, 2)])
def test_many_rows_give_the_same_every_time(N, M, k, dtype):
    """Rows that are streamed through shared memory: a copy that overtakes the loads of
    the last piece would show in some of the runs."""
    C, g, _, ma, mb = (v.cuda() for v in make(1, N, M, TYPES[dtype], N + M))
    first = _skb().row_logprobs(C, g, 0.25, None, k, ma, mb)
    rows = slice(0, None, 97)
    ref = plain(shaped(C[:, rows].cpu(), g.cpu(), ma[:, rows].cpu(), mb.cpu()), 4.0, k=k)
    sub = type(first)(*(None if v is None else v[:, rows] for v in (
        first.lse, first.entropy, first.logprob, first.top_logprob, first.top_index)))
    check(sub, ref, M, k)
    for _ in range(20):
        r = _skb().row_logprobs(C, g, 0.25, None, k, ma, mb)
        assert torch.equal(r.lse, first.lse) and torch.equal(r.entropy, first.entropy)
        assert k == 0 or torch.equal(r.top_index, first.top_index)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", [9, 700, 30000])
def test_masks_of_the_types_lowest_value(V, dtype):
    """Logits masked by the lowest finite value, some rows wholly so: those are uniform."""
    low = torch.finfo(TYPES[dtype]).min
    x = torch.randn(3, V, generator=torch.Generator().manual_seed(V)).to(TYPES[dtype])
    x[0, ::2] = low
    x[1] = low
    X = x.cuda().requires_grad_()
    r = _skb().token_logprobs(X, torch.tensor([1, 2, 3]).cuda(), 4)
    # (shifted by each row's maximum: log 1e4 beside 1e38 is lost in 64 bits, too)
    ref = plain(x.double() - x.double().amax(1, keepdim=True), 1.0, torch.tensor([1, 2, 3]), 4)
    for got, want in ((r.entropy, ref["entropy"]), (r.logprob, ref["logprob"])):
        assert (got.detach().double().cpu() - want).abs().max() < 1e-4
    assert torch.equal(r.top_index.cpu(), ref["top_index"])
    d, = torch.autograd.grad(r.logprob.sum(), X)
    p = ref["p"]
    p[torch.arange(3), torch.tensor([1, 2, 3])] -= 1
    assert (d.double().cpu() + p).abs().max() < torch.finfo(TYPES[dtype]).eps


def test_same_result_twice_and_under_capture_on_another_stream():
    C, g, t, _, mb = make(2, 700, 200, torch.float32, 8)
    t, mb = t.cuda(), mb.cuda()

    def step(X, G):
        r = _skb().row_logprobs(X, G, 0.5, t, 3, None, mb)
        d = torch.autograd.grad(r.logprob.sum() + r.top_logprob.sum() + r.entropy.sum(), (X, G))
        return tuple(v.detach() for v in (r.lse, r.entropy, r.logprob, r.top_index,
                                          r.top_logprob) + d)

    def leaves(scale=1.0):
        return (scale * C).cuda().requires_grad_(), g.cuda().requires_grad_()

    first = step(*leaves())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for v, w in zip(step(*leaves()), first):
            assert torch.equal(v, w)
        held = leaves()  # leaves that no eager graph refers to
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = step(*held)
    torch.cuda.synchronize()
    with torch.no_grad():
        held[0].copy_(2 * C)
    graph.replay()
    torch.cuda.synchronize()
    for v, w in zip(step(*leaves(2.0)), out):
        assert torch.equal(v, w)


@pytest.mark.parametrize("bad", [math.nan, -math.inf, math.inf])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,N,M,k", [(2, 9, 5, 2), (1, 70, 64, 2), (2, 33, 203, 4), (1, 20, 512, 0),
                                     (2, 6, 1031, 5), (1, 5, 9001, 3)])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("aligned", [True, False])
def test_what_a_masked_row_holds_reaches_no_gradient(B, N, M, k, dtype, bad, masked, aligned):
    """The same bits as with zeros in the rows that mask_a leaves out, and zeros there."""
    C, g, t, ma, mb = make(B, N, M, TYPES[dtype], M + k)
    ma[:, 1], ma[:, 0] = False, True
    mb[:, 0] = True
    gen = torch.Generator().manual_seed(3)
    ups = [torch.randn(s, generator=gen).cuda() for s in ((B, N),) * 3 + ((B, N, k),)]
    got = []
    for fill in (0.0, bad):
        Y = C.masked_fill(~ma[..., None], fill)
        X = Y.cuda() if aligned else torch.nn.functional.pad(Y, (1, 2)).cuda()[..., 1:M + 1]
        X, G = X.detach().requires_grad_(), g.cuda().requires_grad_()
        r = _skb().row_logprobs(X, G, 0.5, t.cuda(), k, ma.cuda(), mb.cuda() if masked else None)
        outs = (r.lse, r.logprob, r.entropy) + ((r.top_logprob,) if k else ())
        both = torch.autograd.grad(outs, (X, G), ups[:len(outs)], retain_graph=True)
        alone, = torch.autograd.grad(outs, (G,), ups[:len(outs)])
        # without dg the rows' vectors start elsewhere
        r = _skb().row_logprobs(X, g.cuda(), 0.5, t.cuda(), k, ma.cuda(),
                                mb.cuda() if masked else None)
        outs = (r.lse, r.logprob, r.entropy) + ((r.top_logprob,) if k else ())
        got.append([v.detach() for v in outs]
                   + [*both, alone, *torch.autograd.grad(outs, (X,), ups[:len(outs)])])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    for d in (got[1][len(outs)], got[1][-1]):
        assert torch.isfinite(d).all() and (d.cpu()[~ma] == 0).all() and (d.cpu()[ma] != 0).any()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", [40, 333, 3001, 70000])
def test_rows_that_nothing_is_asked_of_pass_nothing(V, dtype):
    """Positions without a token whose logits are garbage, as behind the end of a padded
    batch: no gradient, and the same bits elsewhere."""
    x = torch.randn(7, V, generator=torch.Generator().manual_seed(V)).to(TYPES[dtype])
    t = torch.tensor([3, -100, 1, -1, 2, -100, 0])
    none = t < 0
    y = x.clone()
    y[1], y[3], y[5, V // 2] = math.nan, math.inf, math.nan
    got = []
    for v in (x, y):
        X = v.cuda().requires_grad_()
        r = _skb().token_logprobs(X, t.cuda(), 3)
        up = torch.where(none, 0.0, 0.5).cuda()
        d1, = torch.autograd.grad(r.logprob.sum(), X, retain_graph=True)
        d2, = torch.autograd.grad((r.logprob, r.entropy, r.lse, r.top_logprob), X,
                                  (torch.ones_like(up), up, up, up[:, None].expand(7, 3)))
        got.append((r.logprob.detach(), d1, d2))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert all((d[none] == 0).all() and (d[~none] != 0).any() for d in got[1][1:])


def test_rows_whose_alternatives_cancel_still_pass_their_gradients():
    x = torch.randn(2, 50, generator=torch.Generator().manual_seed(6))
    X = x.cuda().requires_grad_()
    r = _skb().token_logprobs(X, top_k=2)
    d, = torch.autograd.grad(r.top_logprob, X, torch.tensor([[1.0, -1.0], [0.0, 0.0]]).cuda())
    want = torch.zeros(2, 50)
    i = x[0].topk(2).indices
    want[0, i[0]], want[0, i[1]] = 1.0, -1.0
    assert torch.equal(d.cpu(), want)


def _on_host(ref):
    return {name: v.cpu() for name, v in ref.items()}


@pytest.mark.parametrize("dtype,V", [("fp32", 515), ("fp32", 1999), ("fp32", 4091), ("bf16", 1999),
                                     ("bf16", 4096), ("bf16", 8190), ("fp16", 1031),
                                     ("fp16", 8190)])
@pytest.mark.parametrize("k", [0, 3, 20])
def test_many_rows_of_logits(dtype, V, k):
    """Rows that are streamed without a potential, on 16 bytes and off it."""
    T = 2500
    base = 3 * torch.randn(T, V + 3, generator=torch.Generator().manual_seed(V + k))
    base = base.to(TYPES[dtype]).cuda()
    t = torch.randint(-1, V, (T,), generator=torch.Generator().manual_seed(k))
    for x in (base[:, :V].contiguous(), base[:, 1:V + 1]):
        r = _skb().token_logprobs(x, t.cuda(), k, temperature=0.7)
        check(r, _on_host(plain(x.double(), 1 / 0.7, t.cuda(), k)), V, k)


@pytest.mark.parametrize("dtype,B,N,M", [
    ("fp32", 5, 701, 700), ("fp32", 5, 701, 4091), ("bf16", 5, 701, 1999), ("fp16", 5, 701, 8190),
    ("fp32", 5, 701, 5003), ("bf16", 5, 701, 9001), ("fp16", 7, 97, 8500),  # four warps a row
    ("fp32", 3, 257, 16500), ("bf16", 3, 257, 17001),                        # g not staged
])
@pytest.mark.parametrize("k", [0, 3, 20])
@pytest.mark.parametrize("masked", [False, True])
def test_many_rows_of_several_items(dtype, B, N, M, k, masked):
    """A CTA's run of rows crosses items, each with its own g and masks."""
    C, g, t, ma, mb = (v.cuda() for v in make(B, N, M, TYPES[dtype], M + k))
    if not masked:
        ma = mb = None
    r = _skb().row_logprobs(C, g, 0.25, t, k, ma, mb)
    check(r, _on_host(plain(shaped(C, g, ma, mb), 4.0, t.reshape(-1), k)), M, k)
