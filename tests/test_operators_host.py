"""Refusals of the row, expert and grouped operators, without a GPU: the Python checks on
CPU tensors, and the C entry points on bad problems, pointers and workspaces (pointers are
never dereferenced)."""

from __future__ import annotations

import pytest
import torch

import sinkhorn_b200 as skb

_P = 1 << 20    # an aligned, non-NULL pointer that is never read
_W = 1 << 40
ARG, LAYOUT, WS = 1, 2, 3
F = torch.zeros


def _cases():
    C = F(2, 3, 4)
    i64 = torch.int64
    bf = torch.bfloat16
    d = skb.ExpertDispatch(F(4, dtype=torch.int32), F(2, 2, dtype=torch.int32),
                           F(3, dtype=torch.int32))
    return [
        ("cost on the CPU", lambda: skb.row_logprobs(C), RuntimeError, "no CPU fallback"),
        ("cost 2D", lambda: skb.row_logprobs(F(3, 4)), ValueError, "3D"),
        ("cost float64", lambda: skb.row_logprobs(C.double()), TypeError, "float32"),
        ("cost no tensor", lambda: skb.row_logprobs([1.0]), TypeError, "Tensor"),
        ("logits on the CPU", lambda: skb.token_logprobs(F(3, 4)), RuntimeError, "no CPU"),
        ("logits integers", lambda: skb.token_logprobs(F(3, 4, dtype=i64)), TypeError, "float32"),
        ("logits 0D", lambda: skb.token_logprobs(F(())), ValueError, "vocabulary"),
        ("logits no tensor", lambda: skb.token_logprobs(None), TypeError, "Tensor"),
        ("index float", lambda: skb.expert_dispatch(F(2, 2), 4), RuntimeError, "no CPU"),
        ("index 1D", lambda: skb.expert_dispatch(F(2, dtype=i64), 4), ValueError, "2D"),
        ("no experts", lambda: skb.expert_dispatch(F(2, 2, dtype=i64), 0), ValueError, "between"),
        ("many experts", lambda: skb.expert_dispatch(F(2, 2, dtype=i64), 1025), ValueError,
         "1024"),
        ("experts float", lambda: skb.expert_dispatch(F(2, 2, dtype=i64), 4.0), TypeError, "int"),
        ("rows on the CPU", lambda: skb.dispatch_rows(F(2, 8), d), RuntimeError, "no CPU"),
        ("combine on the CPU", lambda: skb.combine_rows(F(4, 8), d), RuntimeError, "no CPU"),
        ("product on the CPU", lambda: skb.grouped_matmul(F(4, 8, dtype=bf), F(2, 8, 8, dtype=bf),
                                                          F(3, dtype=torch.int32)),
         RuntimeError, "no CPU"),
        ("scores 3D", lambda: skb.sinkhorn_route(C), ValueError, "2D"),
        ("scores on the CPU", lambda: skb.sinkhorn_route(F(3, 4)), RuntimeError, "no CPU"),
        ("layer on the CPU", lambda: skb.sinkhorn_experts(F(3, 4), F(3, 2), F(2, 4, 4),
                                                          F(2, 4, 4)), RuntimeError, "no CPU"),
    ]


@pytest.mark.parametrize("case", _cases(), ids=lambda c: c[0])
def test_python_refusals_without_a_device(case):
    _, call, error, text = case
    with pytest.raises(error, match=text):
        call()


class _Cuda(torch.Tensor):
    """A CPU tensor that says it is on a GPU: the argument checks run, nothing else."""

    @property
    def is_cuda(self):
        return True


def _on(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Cuda)


def _checked():
    i32, i64, bf = torch.int32, torch.int64, torch.bfloat16
    C, L = _on(2, 3, 4), _on(5, 40)
    d = skb.ExpertDispatch(_on(6, dtype=i32), _on(3, 2, dtype=i32), _on(5, dtype=i32))
    x, w, o = _on(6, 8, dtype=bf), _on(2, 8, 4, dtype=bf), _on(3, dtype=i32)
    g = skb.grouped_matmul
    x16 = _on(3, 8, dtype=bf)

    def layer(x, w_in=None, w_out=None):
        w_in = _on(4, 8, 6, dtype=bf) if w_in is None else w_in
        w_out = _on(4, 6, 8, dtype=bf) if w_out is None else w_out
        return skb.sinkhorn_experts(x, _on(3, 4), w_in, w_out)

    return [
        ("top_k", lambda: skb.row_logprobs(C, top_k=5), ValueError, "top_k"),
        ("top_k 33", lambda: skb.token_logprobs(L, top_k=33), ValueError, "32"),
        ("top_k negative", lambda: skb.token_logprobs(L, top_k=-1), ValueError, "top_k"),
        ("top_k float", lambda: skb.token_logprobs(L, top_k=2.0), TypeError, "int"),
        ("top_k bool", lambda: skb.token_logprobs(L, top_k=True), TypeError, "int"),
        ("epsilon 0", lambda: skb.row_logprobs(C, epsilon=0.0), ValueError, "epsilon"),
        ("epsilon nan", lambda: skb.row_logprobs(C, epsilon=float("nan")), ValueError, "epsilon"),
        ("temperature inf", lambda: skb.token_logprobs(L, temperature=float("inf")), ValueError,
         "temperature"),
        ("g shape", lambda: skb.row_logprobs(C, _on(2, 3)), ValueError, "shape"),
        ("g integers", lambda: skb.row_logprobs(C, _on(2, 4, dtype=i64)), TypeError, "floating"),
        ("targets shape", lambda: skb.row_logprobs(C, targets=_on(2, 4, dtype=i64)), ValueError,
         "shape"),
        ("targets float", lambda: skb.token_logprobs(L, _on(5)), TypeError, "integers"),
        ("mask shape", lambda: skb.row_logprobs(C, mask_b=_on(2, 3, dtype=torch.bool)),
         ValueError, "shape"),
        ("no columns", lambda: skb.row_logprobs(_on(2, 3, 0)), ValueError, "columns"),
        ("no vocabulary", lambda: skb.token_logprobs(_on(3, 0)), ValueError, "vocabulary"),
        ("index float", lambda: skb.expert_dispatch(_on(2, 2), 4), TypeError, "integers"),
        ("rows count", lambda: skb.dispatch_rows(_on(4, 8), d), ValueError, "rows"),
        ("rows 1D", lambda: skb.dispatch_rows(_on(3), d), ValueError, "2D"),
        ("rows type", lambda: skb.dispatch_rows(_on(3, 8, dtype=i32), d), TypeError, "float32"),
        ("no plan", lambda: skb.dispatch_rows(_on(3, 8), (1, 2, 3)), TypeError, "ExpertDispatch"),
        ("plan type", lambda: skb.dispatch_rows(_on(3, 8), skb.ExpertDispatch(
            _on(6, dtype=i64), d.position, d.offsets)), TypeError, "int32"),
        ("plan shape", lambda: skb.dispatch_rows(_on(3, 8), skb.ExpertDispatch(
            _on(5, dtype=i32), d.position, d.offsets)), ValueError, "position"),
        ("plan strided", lambda: skb.combine_rows(_on(6, 8), skb.ExpertDispatch(
            d.order, _on(2, 3, dtype=i32).t(), d.offsets)), ValueError, "contiguous"),
        ("weights shape", lambda: skb.combine_rows(_on(6, 8), d, _on(2, 3)), ValueError, "shape"),
        ("weights integers", lambda: skb.combine_rows(_on(6, 8), d, _on(3, 2, dtype=i32)),
         TypeError, "floating"),
        ("product fp32", lambda: g(_on(6, 8), _on(2, 8, 4), o), TypeError, "bfloat16"),
        ("product types", lambda: g(x, _on(2, 8, 4, dtype=torch.float16), o), TypeError, "one"),
        ("product widths", lambda: g(x, _on(2, 9, 4, dtype=bf), o), ValueError, "columns"),
        ("product 2D weights", lambda: g(x, _on(8, 4, dtype=bf), o), ValueError, "3D"),
        ("product offsets", lambda: g(x, w, _on(4, dtype=i32)), ValueError, "offsets"),
        ("product offsets type", lambda: g(x, w, _on(3)), TypeError, "offsets"),
        ("product offsets none", lambda: g(x, w, None), TypeError, "offsets"),
        ("product groups", lambda: g(x, _on(1025, 8, 4, dtype=bf), _on(1026, dtype=i32)),
         ValueError, "1024"),
        ("route top_k", lambda: skb.sinkhorn_route(_on(3, 4), 5), ValueError, "top_k"),
        ("route mask", lambda: skb.sinkhorn_route(_on(3, 4), 1, mask=_on(4, dtype=torch.bool)),
         ValueError, "mask"),
        ("route empty", lambda: skb.sinkhorn_route(_on(0, 4)), ValueError, "at least one"),
        ("route width", lambda: skb.sinkhorn_route(_on(3, 1025)), ValueError, "1024"),
        ("route many", lambda: skb.sinkhorn_route(_on(3, 64), 33), ValueError, "top_k"),
        ("route mask list", lambda: skb.sinkhorn_route(_on(3, 4), 1, mask=[1, 1, 1]), TypeError,
         "mask"),
        ("layer types", lambda: layer(_on(3, 8)), TypeError, "x must be"),
        ("layer mixed", lambda: layer(x16, w_in=_on(4, 8, 6, dtype=torch.float16)), TypeError,
         "one type"),
        ("layer weights", lambda: layer(x16, w_out=[1]), TypeError, "w_out"),
        ("layer weights 2D", lambda: layer(x16, w_in=_on(8, 6, dtype=bf)), ValueError, "3D"),
        ("layer rows", lambda: layer(_on(2, 8, dtype=bf)), ValueError, "3 rows"),
        ("layer experts", lambda: layer(x16, w_out=_on(5, 6, 8, dtype=bf)), ValueError,
         "4 experts"),
        ("layer width", lambda: layer(_on(3, 7, dtype=bf)), ValueError, "7 columns"),
    ]


@pytest.mark.parametrize("case", _checked(), ids=lambda c: c[0])
def test_argument_checks(case):
    _, call, error, text = case
    with pytest.raises(error, match=text):
        call()


def _rows(L, X=_P, dt=0, B=1, N=4, M=8, sb=32, sn=8, sm=1, eps=1.0, mb=None, t=None, k=0,
          lp=None, tl=None, ti=None, ws=None, wsb=0):
    return L.sk_row_logprobs(X, dt, B, N, M, sb, sn, sm, None, eps, 1, None, mb, t, k, _P, lp, _P,
                             tl, ti, None, ws, wsb, None)


def _rows_bwd(L, X=_P, stats=_P, t=None, k=0, ti=None, ent=None, glp=None, gent=None, gtop=None,
              dX=_P, dg=None, ws=None, wsb=0, mb=None):
    return L.sk_row_logprobs_backward(X, 0, 1, 4, 8, 32, 8, 1, None, 1.0, 1, mb, t, k, ti, stats,
                                      ent, None, glp, gent, gtop, dX, dg, ws, wsb, None)


def _gmm(L, x=_P, dt=1, S=16, K=64, ldx=64, w=_P, E=2, N=32, se=2048, sk=32, sn=1, o=_P, y=_P):
    return L.sk_grouped_matmul(x, dt, S, K, ldx, w, E, N, se, sk, sn, o, y, None)


def _gmw(L, x=_P, dt=1, S=16, K=64, ldx=64, dy=_P, N=32, ldy=32, o=_P, E=2, dw=_P):
    return L.sk_grouped_matmul_weight(x, dt, S, K, ldx, dy, N, ldy, o, E, dw, 0, None)


_ENTRIES = [
    ("rows X=NULL", lambda L: _rows(L, X=None), ARG),
    ("rows type", lambda L: _rows(L, dt=3), ARG),
    ("rows M=0", lambda L: _rows(L, M=0), ARG),
    ("rows eps", lambda L: _rows(L, eps=float("inf")), ARG),
    ("rows eps tiny", lambda L: _rows(L, eps=1e-45), ARG),
    ("rows strided columns", lambda L: _rows(L, sm=2), LAYOUT),
    ("rows negative stride", lambda L: _rows(L, sn=-8), LAYOUT),
    ("rows misaligned", lambda L: _rows(L, X=_P + 2), LAYOUT),
    ("rows top_k", lambda L: _rows(L, k=9, tl=_P, ti=_P), ARG),
    ("rows top without outputs", lambda L: _rows(L, k=2, tl=_P), ARG),
    ("rows targets without output", lambda L: _rows(L, t=_P), ARG),
    ("rows output without targets", lambda L: _rows(L, lp=_P), ARG),
    ("rows mask without workspace", lambda L: _rows(L, M=16385, sn=16385, mb=_P), WS),
    ("rows mask, odd workspace", lambda L: _rows(L, M=16385, sn=16385, mb=_P, ws=_P + 4,
                                                 wsb=_W), WS),
    ("rows backward stats=NULL", lambda L: _rows_bwd(L, stats=None), ARG),
    ("rows backward no target", lambda L: _rows_bwd(L, glp=_P), ARG),
    ("rows backward no entropy", lambda L: _rows_bwd(L, gent=_P), ARG),
    ("rows backward no index", lambda L: _rows_bwd(L, gtop=_P, k=2), ARG),
    ("rows backward nothing asked", lambda L: _rows_bwd(L, dX=None), ARG),
    ("rows backward dX misaligned", lambda L: _rows_bwd(L, dX=_P + 8), LAYOUT),
    ("rows backward dg without workspace", lambda L: _rows_bwd(L, dg=_P), WS),
    ("rows backward mask without workspace", lambda L: _rows_bwd(L, mb=_P), WS),
    ("sort index=NULL", lambda L: L.sk_expert_dispatch(None, 4, 2, _P, _P, _P, _P, _W, None), ARG),
    ("sort no slots", lambda L: L.sk_expert_dispatch(_P, 0, 2, _P, _P, _P, _P, _W, None), ARG),
    ("sort 1025 experts", lambda L: L.sk_expert_dispatch(_P, 4, 1025, _P, _P, _P, _P, _W, None),
     ARG),
    ("sort no workspace", lambda L: L.sk_expert_dispatch(_P, 2049, 2, _P, _P, _P, None, 0, None),
     WS),
    ("dispatch x=NULL", lambda L: L.sk_dispatch_rows(None, 1, 4, 2, 8, 8, _P, _P, 2, _P, None),
     ARG),
    ("dispatch T k", lambda L: L.sk_dispatch_rows(_P, 1, 1 << 30, 4, 8, 8, _P, _P, 2, _P, None),
     ARG),
    ("dispatch odd address", lambda L: L.sk_dispatch_rows(_P + 1, 1, 4, 2, 8, 8, _P, _P, 2, _P,
                                                          None), LAYOUT),
    ("dispatch fp32 on 2 bytes", lambda L: L.sk_dispatch_rows(_P + 2, 0, 4, 2, 8, 8, _P, _P, 2,
                                                              _P, None), LAYOUT),
    ("combine out=NULL", lambda L: L.sk_combine_rows(_P, 1, 4, 2, 8, 8, _P, _P, 2, None, None,
                                                     None), ARG),
    ("combine stride", lambda L: L.sk_combine_rows(_P, 1, 4, 2, 8, -8, _P, _P, 2, None, _P,
                                                   None), LAYOUT),
    ("combine position=NULL", lambda L: L.sk_combine_rows(_P, 1, 4, 2, 8, 8, None, _P, 2, None,
                                                          _P, None), ARG),
    ("combine backward nothing asked", lambda L: L.sk_combine_rows_backward(
        _P, _P, 1, 4, 2, 8, 8, 8, _P, _P, 2, _P, None, None, None), ARG),
    ("combine backward y=NULL", lambda L: L.sk_combine_rows_backward(
        _P, None, 1, 4, 2, 8, 8, 8, _P, _P, 2, _P, None, _P, None), ARG),
    ("product fp32", lambda L: _gmm(L, dt=0), ARG),
    ("product S=0", lambda L: _gmm(L, S=0), ARG),
    ("product E=1025", lambda L: _gmm(L, E=1025), ARG),
    ("product offsets=NULL", lambda L: _gmm(L, o=None), ARG),
    ("product y=NULL", lambda L: _gmm(L, y=None), ARG),
    ("product weights without a unit stride", lambda L: _gmm(L, sk=64, sn=2), LAYOUT),
    ("product negative stride", lambda L: _gmm(L, ldx=-64), LAYOUT),
    ("product unaligned stride", lambda L: _gmm(L, ldx=65), LAYOUT),
    ("product unaligned address", lambda L: _gmm(L, w=_P + 2), LAYOUT),
    ("product overlapping rows", lambda L: _gmm(L, ldx=0), LAYOUT),
    ("pack src=NULL", lambda L: L.sk_grouped_pack(None, 1, 4, 7, 28, 7, _P, None), ARG),
    ("pack no rows", lambda L: L.sk_grouped_pack(_P, 1, 0, 7, 28, 7, _P, None), ARG),
    ("pack rows", lambda L: L.sk_grouped_pack(_P, 1 << 20, 1 << 20, 7, 28, 7, _P, None), ARG),
    ("pack stride", lambda L: L.sk_grouped_pack(_P, 1, 4, 7, 28, -7, _P, None), LAYOUT),
    ("pack dst", lambda L: L.sk_grouped_pack(_P, 1, 4, 7, 28, 7, _P + 8, None), LAYOUT),
    ("product too many tiles", lambda L: _gmm(L, S=1 << 30, K=8, N=1 << 20, sk=1 << 20,
                                              se=1 << 23), ARG),
    ("weight product dw=NULL", lambda L: _gmw(L, dw=None), ARG),
    ("weight product unaligned", lambda L: _gmw(L, ldy=33), LAYOUT),
]


@pytest.mark.parametrize("case", _ENTRIES, ids=lambda c: c[0])
def test_entry_points_reject_bad_arguments_without_a_device(case):
    from sinkhorn_b200 import _lib
    lib = _lib.load()
    _, call, code = case
    assert call(lib) == code, lib.sk_last_error()
    assert lib.sk_last_error().decode()


def test_workspace_sizes():
    from sinkhorn_b200 import _lib
    L = _lib.load()
    assert L.sk_row_logprobs_workspace_bytes(4, 16384) == 0
    assert L.sk_row_logprobs_workspace_bytes(4, 16385) >= 4 * 4 * 16385
    assert L.sk_row_logprobs_backward_workspace_bytes(0, 8, 8) == 0
    assert L.sk_row_logprobs_backward_workspace_bytes(2, 100, 64) >= 2 * 4 * 2 * 64
    assert L.sk_expert_dispatch_workspace_bytes(2048, 8) == 0
    assert L.sk_expert_dispatch_workspace_bytes(5000, 8) >= 3 * 8 * 4


def test_public_names():
    for name in ("row_logprobs", "token_logprobs", "RowLogprobs", "expert_dispatch",
                 "dispatch_rows", "combine_rows", "ExpertDispatch", "grouped_matmul",
                 "sinkhorn_route", "sinkhorn_experts", "Route"):
        assert hasattr(skb, name) and name in skb.__all__
    assert hasattr(skb.SinkhornOutput, "assign")


@pytest.mark.parametrize("call", [
    lambda L, o, p: L.sk_dispatch_plan_rows(_P, 1, 4, 2, 8, 8, o, p, _P, 2, _P, None),
    lambda L, o, p: L.sk_combine_plan_rows(_P, 1, 4, 2, 8, 8, o, p, _P, 2, None, _P, None),
    lambda L, o, p: L.sk_combine_plan_rows_backward(_P, _P, 1, 4, 2, 8, 8, 8, o, p, _P, 2, None,
                                                    _P, None, None),
], ids=["dispatch", "combine", "backward"])
def test_calls_with_a_plan_need_its_order_and_positions(call):
    from sinkhorn_b200 import _lib
    lib = _lib.load()
    for order, position in ((None, _P), (_P, None)):
        assert call(lib, order, position) == ARG and lib.sk_last_error().decode()


def test_the_sorts_counts_do_not_grow_with_the_slots():
    """Every CTA of the sort adds up all counts: few, whatever the slots, or its work would
    grow with their square."""
    from sinkhorn_b200 import _lib
    L = _lib.load()
    for experts in (1, 256, 1024):
        most = L.sk_expert_dispatch_workspace_bytes(2 ** 31 - 1, experts)
        assert 0 < most <= 4 * 1024 * experts + 256
        assert most >= L.sk_expert_dispatch_workspace_bytes(1 << 20, experts)
