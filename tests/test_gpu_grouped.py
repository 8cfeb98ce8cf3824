"""Products grouped by expert over ragged runs of rows, with both gradients, against
plain products in 64 bits.

Inputs are bf16 or fp16, so their products are exact in fp32; a sum of n of them in fp32 is
off by at most n u sum|x w| (u = 2^-24, any order; the tensor core's own adders keep at
least that when u is doubled), and the result is rounded once to the type.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _gmm(*a):
    import sinkhorn_b200
    return sinkhorn_b200.grouped_matmul(*a)


def close(got, want, size, n):
    """want and the sum of absolute products `size`, both fp64."""
    t = torch.finfo(got.dtype)
    bound = t.eps / 2 * want.abs() + 2 * n * U32 * size + t.tiny
    off = (got.detach().double().cpu() - want).abs()
    assert (off <= bound).all(), float((off - bound).max())


def plain(x, w, ends):
    y, a = (torch.zeros(x.shape[0], w.shape[2], dtype=torch.float64) for _ in range(2))
    for e in range(w.shape[0]):
        r = slice(ends[e], ends[e + 1])
        y[r] = x[r].double() @ w[e].double()
        a[r] = x[r].double().abs() @ w[e].double().abs()
    return y, a


def check(x, w, ends, grads=True, seed=0):
    """x, w on the GPU (any layout)."""
    offsets = torch.tensor(ends, dtype=torch.int32).cuda()
    X, W = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = _gmm(X, W, offsets)
    x, w = x.cpu(), w.cpu()
    want, size = plain(x, w, ends)
    close(y, want, size, x.shape[1])
    if not grads:
        return
    g = torch.randn(y.shape, generator=torch.Generator().manual_seed(seed)).to(y.dtype)
    dx, dw = torch.autograd.grad(y, (X, W), g.cuda())
    want, size = plain(g, w.transpose(1, 2), ends)
    close(dx, want, size, w.shape[2])
    assert dw.shape == w.shape
    for e in range(w.shape[0]):
        r = slice(ends[e], ends[e + 1])
        close(dw[e], x[r].double().T @ g[r].double(), x[r].double().abs().T @ g[r].double().abs(),
              max(1, ends[e + 1] - ends[e]))


def make(S, E, K, N, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(S, K, generator=gen).to(TYPES[dtype]).cuda(),
            (torch.randn(E, K, N, generator=gen) / K ** 0.5).to(TYPES[dtype]).cuda())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("S,E,K,N,ends", [
    (16, 1, 64, 128, [0, 16]),
    (1, 1, 8, 8, [0, 1]),
    (128, 1, 128, 256, [0, 128]),
    (300, 2, 192, 136, [0, 44, 300]),
    (300, 3, 72, 40, [0, 0, 299, 299]),          # empty groups, a row of no group
    (700, 5, 264, 520, [3, 10, 257, 257, 530, 690]),  # rows before and behind the groups
    (520, 4, 64, 64, [0, 1, 17, 33, 520]),
    (1100, 2, 320, 128, [0, 550, 1100]),
    (2000, 40, 128, 128, [50 * i for i in range(41)]),
    (64, 3, 4096, 24, [0, 20, 40, 64]),
])
def test_products_and_gradients(S, E, K, N, ends, dtype):
    check(*make(S, E, K, N, dtype, S + K), ends)


@pytest.mark.parametrize("K,N", [(1, 1), (1, 40), (40, 1), (1, 7), (9, 1), (16, 1), (7, 3), (33, 65), (64, 77), (1001, 64), (130, 262)])
def test_widths_that_are_not_multiples_of_eight(K, N):
    check(*make(150, 3, K, N, "bf16", K), [0, 70, 71, 149])
    check(*make(90, 2, K, N, "fp16", K), [0, 33, 90])


@pytest.mark.parametrize("E", [31, 32, 33, 200, 1024])
def test_many_groups(E):
    gen = torch.Generator().manual_seed(E)
    lengths = torch.randint(0, 9, (E,), generator=gen)
    ends = [0] + lengths.cumsum(0).tolist()
    check(*make(ends[-1] + 5, E, 40, 16, "bf16", E), ends)


def test_no_rows_at_all():
    x, w = make(0, 2, 16, 24, "bf16")
    X, W = x.requires_grad_(), w.requires_grad_()
    y = _gmm(X, W, torch.tensor([0, 0, 0]).cuda())
    dx, dw = torch.autograd.grad(y.sum(), (X, W))
    assert y.shape == (0, 24) and dx.shape == (0, 16) and (dw == 0).all()
    check(*make(37, 2, 16, 24, "bf16"), [0, 0, 0])
    check(*make(37, 2, 16, 24, "bf16"), [37, 37, 37])


@pytest.mark.parametrize("layout", ["transposed", "sliced", "offset", "expanded", "strided"])
def test_layouts(layout):
    gen = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen).bfloat16().cuda()
    ends = [0, 100, 131, 200]
    x, w = r(200, 96), r(3, 96, 72)
    if layout == "transposed":
        w = r(3, 72, 96).transpose(1, 2)
        W = w.detach().requires_grad_()
        y = _gmm(x, W, torch.tensor(ends).cuda())
        dw, = torch.autograd.grad(y.float().sum(), W)
        assert dw.stride() == w.stride()
    elif layout == "sliced":
        x, w = r(200, 200)[:, 8:104], r(6, 96, 144)[::2, :, 16:88]
    elif layout == "offset":  # rows off the 16-byte grid
        x, w = r(200, 97)[:, 1:], r(3, 96, 73)[:, :, 1:]
    elif layout == "expanded":
        x, w = r(1, 96).expand(200, 96), r(1, 96, 72).expand(3, 96, 72)
    else:
        x, w = r(96, 200).t(), r(3, 96, 144)[:, :, ::2]
    check(x, w, ends)


@pytest.mark.parametrize("what", ["nan", "inf"])
def test_what_is_in_other_groups_stays_there(what):
    """NaN and infinities in one group's rows or weights reach no other group."""
    v = float(what)
    x, w = make(210, 3, 72, 88, "bf16", 5)
    ends = [0, 37, 150, 200]
    x[37:150] = v
    x[200:] = v
    w[1] = v
    g = torch.randn(210, 88, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    g[37:150] = v
    g[200:] = v
    X, W = x.requires_grad_(), w.requires_grad_()
    y = _gmm(X, W, torch.tensor(ends).cuda())
    dx, dw = torch.autograd.grad(y, (X, W), g)
    for t in (y, dx):
        assert torch.isfinite(t[:37]).all() and torch.isfinite(t[150:]).all()
        assert (t[200:] == 0).all() and not torch.isfinite(t[37:150]).any()
    assert torch.isfinite(dw[0]).all() and torch.isfinite(dw[2]).all()
    assert not torch.isfinite(dw[1]).any()


def test_offsets_that_fall_or_leave_the_rows_are_clamped():
    x, w = make(100, 3, 64, 64, "bf16", 7)
    y = _gmm(x, w, torch.tensor([-5, 40, 30, 1000]).cuda())
    want = _gmm(x, w, torch.tensor([0, 40, 40, 100]).cuda())
    assert torch.equal(y, want)


def test_gradient_against_differences():
    x, w = make(20, 2, 16, 8, "fp16", 11)
    offsets = torch.tensor([0, 12, 20]).cuda()
    X, W = x.clone().requires_grad_(), w.clone().requires_grad_()
    g = torch.ones(20, 8, device="cuda", dtype=torch.float16)
    dx, dw = torch.autograd.grad(_gmm(X, W, offsets), (X, W), g)
    # the product is linear in each: a difference of step 1 errs by the outputs' rounding alone
    for t, d, at in ((x, dx, (3, 5)), (x, dx, (15, 0)), (w, dw, (0, 2, 3)), (w, dw, (1, 7, 7))):
        up = t.clone()
        up[at] += 1
        step = float(up[at]) - float(t[at])
        a = _gmm(up if t is x else x, up if t is w else w, offsets).double().sum()
        b = _gmm(x, w, offsets).double().sum()
        y = _gmm(x, w, offsets).double().abs()
        bound = 2.0 ** -11 * 3 * float(y.sum() + abs(float(d[at])) * 20) + 2.0 ** -11 * abs(float(d[at]))
        assert abs(float(a - b) / step - float(d[at])) <= bound


def test_int64_offsets_captured_and_replayed_with_other_lengths():
    x, w = make(300, 4, 64, 96, "bf16", 3)
    offsets = torch.tensor([0, 50, 50, 200, 300]).cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _gmm(x, w, offsets)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            y = _gmm(x, w, offsets)
    torch.cuda.synchronize()
    offsets.copy_(torch.tensor([0, 0, 120, 250, 290]).cuda())
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, _gmm(x, w, offsets))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("S,K,N,ends,transposed", [
    (2700, 264, 2100, [0, 2300, 2600], False),   # rows: nine column tiles, nine rows of tiles
    (2700, 520, 328, [5, 100, 2700], True),
    (300, 2100, 520, [0, 130, 290], False),      # weights: nine column tiles, three rows
    (300, 520, 2100, [0, 130, 290], True),
    (4700, 264, 264, [0, 4500, 4700], False),    # two bands and a half
])
def test_tiles_in_several_bands(S, K, N, ends, transposed, dtype):
    x, w = make(S, 2, K, N, dtype, S + K)
    check(x, w.transpose(1, 2).contiguous().transpose(1, 2) if transposed else w, ends)
