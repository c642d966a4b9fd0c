"""CPU checks of what the entry points of the microscaled 4-bit matrices and of the
sorting of tokens by expert refuse, and of the plain forms that their tests use."""
import ctypes as C

import pytest
import torch

import mx4_util as U
from spindle_b200 import _lib, mx4

OK, INVALID, DTYPE, SHAPE, ALIGN = 0, 1, 2, 3, 4
AT = 0x100000  # an address that is never read: every call here is refused before a launch


def mat(rows=64, cols=256, experts=1, data=AT):
    return _lib.SgMx4(experts, rows, cols, data)


def plan(n_tok=4, n_used=2, n_expert=8, **kw):
    at = dict(ids=AT, weights=AT, first=AT, order=AT, place=AT, work=AT)
    at.update(kw)
    return _lib.SgMoePlan(n_tok, n_used, n_expert, *(at[k] for k in ("ids", "weights", "first", "order", "place", "work")))


def test_bytes():
    L = _lib.load()
    tile = 128 * 128 + 1024
    for e, r, c, tiles in ((1, 1, 32, 1), (1, 128, 256, 1), (1, 129, 256, 2), (1, 128, 288, 2), (3, 200, 4096, 3 * 2 * 16)):
        assert L.sg_mx4_bytes(C.byref(mat(r, c, e))) == tiles * tile
    for e, r, c in ((0, 1, 32), (1, 0, 32), (1, 1, 0), (1, 1, 16), (1, 1, 100), (1, 1 << 31, 32), (1 << 24, 128, 32), (1, 1, 1 << 31)):
        assert L.sg_mx4_bytes(C.byref(mat(r, c, e))) == 0
        with pytest.raises(_lib.SgError):
            mx4.Mx4.bytes_for(r, c, e)


@pytest.mark.parametrize("fn", ["sg_mx4_quantize", "sg_mx4_dequantize"])
def test_rows_refusals(fn):
    f = getattr(_lib.load(), fn)
    call = lambda m=mat(), t=0, x=AT, ld=256, le=0: f(C.byref(m), t, x, ld, le, None)  # noqa: E731
    assert f(None, 0, AT, 256, 0, None) == INVALID
    assert call(t=8) == DTYPE and call(t=12) == DTYPE
    assert call(m=mat(cols=100)) == SHAPE
    assert call(m=mat(data=None)) == INVALID and call(m=mat(data=AT + 8)) == ALIGN
    assert call(x=None) == INVALID and call(ld=255) == INVALID
    assert call(x=AT + 2) == ALIGN and call(t=1, x=AT + 1) == ALIGN


def test_product_refusals():
    L = _lib.load()

    def call(w=None, up=None, t=0, x=AT, ldx=256, n=4, ot=0, out=AT, ldo=64, scratch=AT, size=1 << 30):
        w = w or mat()
        return L.sg_mx4_matmul(C.byref(w), None if up is None else C.byref(up), t, x, ldx, n, ot, out, ldo, scratch, size, None)
    assert call(t=8) == DTYPE and call(ot=14) == DTYPE
    assert call(w=mat(experts=2)) == SHAPE and call(up=mat(rows=63)) == SHAPE and call(up=mat(cols=512)) == SHAPE
    assert call(up=mat(data=None)) == INVALID
    assert call(x=None) == INVALID and call(out=None) == INVALID and call(scratch=None) == INVALID
    assert call(ldx=255) == INVALID and call(ldo=63) == INVALID and call(n=1 << 31) == INVALID
    need = L.sg_mx4_scratch_bytes(C.byref(mat()), 40, None)
    assert need > 0 and call(n=40, size=need - 1) == INVALID
    assert call(x=AT + 2) == ALIGN and call(out=AT + 1, ot=1) == ALIGN and call(n=40, scratch=AT + 64) == ALIGN
    assert call(n=0, x=None, out=None, scratch=None) == OK  # nothing to do

    def experts(w=None, p=None, gather=1, n_rows=0, **kw):
        a = dict(t=0, x=AT, ldx=256, ot=0, out=AT, ldo=64, scratch=AT, size=1 << 30)
        a.update(kw)
        return L.sg_mx4_experts(C.byref(w or mat(experts=8)), None, C.byref(p or plan()), a["t"], a["x"], a["ldx"], gather, a["ot"], a["out"],
                                a["ldo"], a["scratch"], a["size"], None)
    assert experts(w=mat(experts=7)) == SHAPE and experts(p=plan(n_used=17)) == SHAPE and experts(p=plan(n_expert=1025)) == SHAPE
    assert experts(p=plan(first=None)) == INVALID and experts(p=plan(order=None)) == INVALID
    assert experts(t=8) == DTYPE and experts(ldx=10) == INVALID and experts(size=0) == INVALID
    assert experts(p=plan(n_tok=0), x=None, out=None, scratch=None) == OK


def test_sort_refusals():
    L = _lib.load()
    route = lambda p=plan(), t=0, x=AT, ld=8: L.sg_moe_route(t, x, ld, 1, 0.0, C.byref(p), None)  # noqa: E731
    assert route(p=plan(n_used=0)) == SHAPE and route(p=plan(n_used=17)) == SHAPE
    assert route(p=plan(n_expert=0)) == SHAPE and route(p=plan(n_expert=1025)) == SHAPE
    assert route(p=plan(n_tok=1 << 30, n_used=2)) == SHAPE
    assert route(t=8) == DTYPE and route(x=None) == INVALID and route(ld=7) == INVALID and route(x=AT + 2) == ALIGN
    for k in ("ids", "weights", "first", "order", "place", "work"):
        assert route(p=plan(**{k: AT + 2})) == ALIGN and L.sg_moe_sort(C.byref(plan(**{k: AT + 2})), None) == ALIGN
        assert route(p=plan(**{k: None})) == INVALID and L.sg_moe_sort(C.byref(plan(**{k: None})), None) == INVALID
    assert L.sg_moe_plan_work_bytes(10, 0) == 0 and L.sg_moe_plan_work_bytes(10, 1025) == 0 and L.sg_moe_plan_work_bytes(10, 8) == 4 * 36
    comb = lambda p=plan(), t=0, y=AT, ldy=64, dim=64, ot=0, o=AT, ldo=64: L.sg_moe_combine(C.byref(p), t, y, ldy, dim, ot, o, ldo, None)  # noqa: E731
    assert comb(t=8) == DTYPE and comb(ot=8) == DTYPE and comb(dim=0) == SHAPE and comb(ldy=63) == INVALID and comb(ldo=63) == INVALID
    assert comb(y=None) == INVALID and comb(o=None) == INVALID and comb(y=AT + 2) == ALIGN
    assert comb(p=plan(n_tok=0), y=None, o=None) == OK
    # 8 rows of y, 4 of out: no byte in common
    assert comb(o=AT + 8 * 256 - 4) == INVALID and comb(o=AT - 4 * 256 + 4) == INVALID


def test_host_tensors():
    with pytest.raises(ValueError):
        mx4.mx4_quantize(torch.zeros(2, 32))
    with pytest.raises(ValueError):
        mx4.Mx4(2, 32, data=torch.zeros(1 << 16, dtype=torch.uint8))


def test_the_plain_quantizer():
    # by hand: a top of 6 keeps its exponent, 7 (1.75 times 4) takes the next one, ties go to the even code
    x = torch.zeros(3, 32)
    x[0, :9] = torch.tensor([6, -5, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -0.2])
    x[1, :5] = torch.tensor([7, 5, 3, 1, -0.5])
    x[2, 0] = float("inf")
    q = U.quantized(x)
    assert q[0, :9].tolist() == [6, -4, 4, 2, 2, 1, 1, 0, 0]
    assert q[1, :5].tolist() == [8, 4, 3, 1, 0]
    assert q[2].isnan().all()
    assert U.quantized(torch.full((1, 32), 2.0 ** -149)).abs().max() == 0 and U.quantized(torch.full((1, 32), 3e38))[0, 0] == 2.0 ** 128


def test_the_plain_choice():
    ids, w = U.choice(torch.tensor([[1.0, 3.0, 3.0, float("-inf")], [float("-inf")] * 4]), 3, True)
    assert ids.tolist() == [[1, 2, 0], [-1, -1, -1]] and abs(w[0].sum() - 1) < 1e-12 and w[1].sum() == 0
    first, order, place = U.sort(torch.tensor([[2, 0], [0, 9], [2, 2]]), 3)
    assert first.tolist() == [0, 2, 2, 5] and order.tolist() == [1, 2, 0, 4, 5, -1] and place.tolist() == [[2, 0], [1, -1], [3, 4]]
