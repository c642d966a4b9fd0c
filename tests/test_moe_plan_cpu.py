"""What a plan of tokens sorted by expert holds after calls that are refused: on the CPU, the
library's answers given by the test (nothing is launched)."""
import ctypes as C

import pytest
import torch

from spindle_b200 import _lib, mx4

INVALID, ALIGN, CUDA = 1, 4, 5


class HostPlan(mx4.MoePlan):
    """A plan in host memory."""

    def __init__(self, max_tokens, n_used, n_expert):
        self.max_tokens, self.n_used, self.n_expert, self.dev = max_tokens, n_used, n_expert, -1
        n = max_tokens * n_used
        self._ids, self._order, self._place = (torch.arange(n, dtype=torch.int32) for _ in range(3))
        self._weights = torch.zeros(n)
        self.desc = _lib.SgMoePlan(0, n_used, n_expert, *[t.data_ptr() for t in (self._ids, self._weights, self._ids, self._order, self._place)], None)
        self._c = C.byref(self.desc)
        self._tokens(0)


@pytest.fixture
def lib(monkeypatch):
    """The library in the place of which every call has the status that the test sets, and the tokens that the calls were
    made for."""
    class Lib:
        status, tokens = 0, []

        def sg_moe_route(self, *a):
            Lib.tokens.append(plan_of(a[5]))
            return Lib.status

        def sg_moe_sort(self, *a):
            Lib.tokens.append(plan_of(a[0]))
            return Lib.status

    def plan_of(ref):
        return ref._obj.n_tok
    Lib.tokens = []
    monkeypatch.setattr(mx4._lib, "load", Lib)
    monkeypatch.setattr(mx4, "_dev", lambda t, what: -1)
    monkeypatch.setattr(mx4, "_s", lambda stream, t: stream and stream.cuda_stream)
    return Lib


def state(p):
    return p.n_tok, p.desc.n_tok, p.ids.tolist(), p.order.tolist(), p.place.tolist(), p.weights.tolist()


def filled(lib, n=6, most=10):
    lib.status = 0
    p = HostPlan(most, 2, 8)
    mx4.moe_sort(torch.full((n, 2), 3, dtype=torch.int32), torch.ones(n, 2), p)
    assert state(p)[:2] == (n, n) and p.ids.shape == (n, 2)
    return p


@pytest.mark.parametrize("n", [3, 9])
def test_a_refused_sort_leaves_the_plan(lib, n):
    ids, w = torch.zeros(n, 2, dtype=torch.int32), torch.zeros(n, 2)
    wrong = [(TypeError, (ids.long(), w)), (TypeError, (torch.zeros(2, n, dtype=torch.int32).T, w)), (ValueError, (ids, w.double())),
             (ValueError, (ids, w[:, :1])), (ValueError, (torch.zeros(11, 2, dtype=torch.int32), torch.zeros(11, 2)))]
    for error, args in wrong:
        p = filled(lib)
        before, calls = state(p), len(lib.tokens)
        with pytest.raises(error):
            mx4.moe_sort(*args, p)
        assert state(p) == before and len(lib.tokens) == calls


@pytest.mark.parametrize("n", [3, 9])
def test_a_refused_route_leaves_the_plan(lib, n):
    p = filled(lib)
    before = state(p)
    for x in (torch.zeros(n, 7), torch.zeros(8, n).T, torch.zeros(11, 8)):
        with pytest.raises(ValueError):
            mx4.moe_route(x, p)
        assert state(p) == before
    with pytest.raises(TypeError):
        mx4.moe_route(torch.zeros(n, 8, dtype=torch.float64), p)
    with pytest.raises(ValueError):
        mx4.moe_route(torch.zeros(n, 8), p, prune="none")
    with pytest.raises(AttributeError):
        mx4.moe_sort(torch.zeros(n, 2, dtype=torch.int32), torch.zeros(n, 2), p, stream="none")
    assert state(p) == before
    for status in (INVALID, ALIGN):  # refused by the library: rows one over the other, or between words
        lib.status = status
        with pytest.raises(_lib.SgError):
            mx4.moe_route(torch.zeros(1, 8).expand(n, 8), p)
        assert lib.tokens[-1] == n and state(p) == before


@pytest.mark.parametrize("n", [3, 9])
def test_a_call_that_failed_leaves_an_empty_plan(lib, n):
    # a launch that failed may have written some of the plan's arrays: it holds no tokens then
    for call in (lambda p: mx4.moe_route(torch.zeros(n, 8), p), lambda p: mx4.moe_sort(torch.zeros(n, 2, dtype=torch.int32), torch.zeros(n, 2), p)):
        p = filled(lib)
        lib.status = CUDA
        with pytest.raises(_lib.SgError):
            call(p)
        assert lib.tokens[-1] == n and p.n_tok == p.desc.n_tok == 0 and p.ids.shape == (0, 2)


def test_calls_set_the_tokens(lib):
    p = filled(lib)
    for n in (9, 0, 3):
        assert mx4.moe_route(torch.zeros(n, 8), p) is p and state(p)[:2] == (n, n) and lib.tokens[-1] == n and p.order.shape == (2 * n,)
        assert mx4.moe_sort(torch.zeros(n, 2, dtype=torch.int32), torch.zeros(n, 2), p) is p and lib.tokens[-1] == n


@pytest.mark.parametrize("e,k,rows,cols", [(1, 1, 100, 64), (8, 2, 300, 512), (60, 6, 129, 1024), (128, 8, 768, 2048), (1000, 16, 40, 96)])
def test_scratch_grows_with_the_tokens(e, k, rows, cols):
    # what is made for the largest step serves every smaller one
    L, m = _lib.load(), _lib.SgMx4(e, rows, cols, None)
    last = 0
    for n in list(range(0, 700)) + list(range(700, 20000, 37)):
        size = L.sg_mx4_scratch_bytes(C.byref(m), 0, C.byref(_lib.SgMoePlan(n, k, e)))
        assert size >= last
        last = size
    one, last = _lib.SgMx4(1, rows, cols, None), 0
    for n in range(0, 3000):
        size = L.sg_mx4_scratch_bytes(C.byref(one), n, None)
        assert size >= last
        last = size


def test_tile_refusals():
    L, many, rows = _lib.load(), C.c_int32(), C.c_int32()
    mat, plan = _lib.SgMx4(8, 64, 256, None), _lib.SgMoePlan(4, 2, 8)
    call = lambda m=mat, n=4, p=None, a=many, b=rows: L.sg_mx4_tile(C.byref(m), 0, n, p and C.byref(p), a and C.byref(a), b and C.byref(b))  # noqa: E731
    assert L.sg_mx4_tile(None, 0, 4, None, C.byref(many), C.byref(rows)) == INVALID
    assert call(a=None) == INVALID and call(b=None) == INVALID and call(n=1 << 31) == INVALID
    assert call(m=_lib.SgMx4(8, 64, 100, None)) == 3
    for p in (_lib.SgMoePlan(4, 0, 8), _lib.SgMoePlan(4, 17, 8), _lib.SgMoePlan(4, 2, 0), _lib.SgMoePlan(1 << 31, 2, 8)):
        assert call(p=p) == 3


def test_sort_of_the_plans_own_arrays(lib):
    # rows of what the plan holds already, in another order or without some
    for pick in (lambda t: t[:3], lambda t: t[2:], lambda t: t[::2], lambda t: t[1:4]):
        p = HostPlan(12, 2, 8)
        ids, w = torch.arange(20, dtype=torch.int32).view(10, 2) % 8, torch.rand(10, 2)
        mx4.moe_sort(ids, w, p)
        mx4.moe_sort(pick(p.ids).contiguous() if pick(p.ids).stride(0) != 2 else pick(p.ids), pick(p.weights), p)
        assert torch.equal(p.ids, pick(ids)) and torch.equal(p.weights, pick(w)) and p.n_tok == pick(ids).shape[0]


def test_read_back_refuses_rows_over_one_another():
    # element (e, r, c) at e * ld_expert + r * ld + c: two experts' would be the same
    L, at = _lib.load(), 0x100000
    call = lambda e, r, ld, le: L.sg_mx4_dequantize(C.byref(_lib.SgMx4(e, r, 64, at)), 0, at, ld, le, None)  # noqa: E731
    for e, r, ld, le in ((2, 4, 64, 0), (2, 4, 64, 255), (2, 4, 100, 63), (3, 4, 191, 64), (3, 1, 64, 63), (2, 4, 128, 100)):
        assert call(e, r, ld, le) == INVALID
