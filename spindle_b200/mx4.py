"""Matrices in microscaled 4 bits, which the tensor cores multiply as they are:
mx4_quantize and mx4_dequantize, products with a few rows or with a prompt's
(mx4_matmul), and a mixture of experts on them: the choice of experts and the tokens
sorted by expert (moe_route, moe_sort), the experts' products (mx4_experts) and the
weighted sum back (moe_combine), through the C ABI (sg_mx4_*, sg_moe_route and
so on).  The reference's K-quant path (matmul_batch, moe_forward_batch) is
another format and stays as it is.

    w = mx4_quantize(weights)                         # once
    y = mx4_matmul(x, w)                              # any number of rows

    plan = MoePlan(max_tokens, n_used, n_expert)
    moe_route(logits, plan)
    h = mx4_experts(x, gate, plan, up=up)             # silu(x gate) * (x up), rows sorted by expert
    y = moe_combine(mx4_experts(h, down, plan), plan)

Everything is device memory; a call can be captured and replayed."""
import ctypes as C

import torch

from . import _lib
from ._lib import SgMoePlan, SgMx4
from .kv4 import _dev, _i32, _on, _s, _type


class Mx4:
    """experts (1: a plain matrix) of rows x cols values in 4 bits, cols a multiple
    of 32.  data: the device bytes (a uint8 CUDA tensor of Mx4.bytes_for), allocated
    if None."""

    def __init__(self, rows, cols, experts=1, device=None, data=None):
        self.rows, self.cols, self.experts = rows, cols, experts
        need = self.bytes_for(rows, cols, experts)
        if data is None:
            data = torch.zeros(need, dtype=torch.uint8, device=device or "cuda")
        if data.dtype != torch.uint8 or not data.is_cuda or not data.is_contiguous() or data.numel() < need:
            raise ValueError("data must be a contiguous uint8 CUDA tensor of %d bytes" % need)
        self.data, self.dev = data, data.get_device()
        self.desc = SgMx4(experts, rows, cols, data.data_ptr())
        self._c = C.byref(self.desc)

    @staticmethod
    def bytes_for(rows, cols, experts=1):
        n = _lib.load().sg_mx4_bytes(C.byref(SgMx4(experts, rows, cols, None)))
        if not n:
            raise _lib.SgError(3, "mx4_bytes")
        return n


def _matrix(m, t, what, dev):
    """Row and expert stride of t, a tensor of m's shape ([rows, cols], or [experts, rows, cols])."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 2:
        rows, cols = shape
        ok, strides = m.experts == 1, (stride[0], 0)
    elif len(shape) == 3:
        experts, rows, cols = shape
        ok, strides = experts == m.experts, (stride[1], stride[0])
    else:
        ok = False
    if not ok or rows != m.rows or cols != m.cols or stride[-1] != 1 or t.get_device() != dev or m.dev != dev:
        raise ValueError("%s must be a tensor of the matrix's shape with contiguous rows on its CUDA device" % what)
    return strides


def mx4_quantize(x, out=None, stream=None):
    """The Mx4 of x [rows, cols] or [experts, rows, cols] (float32, float16 or
    bfloat16, contiguous rows any distance apart), or into out."""
    dev, kind = _dev(x, "x"), _type(x, "x")
    if out is None:
        shape = x.shape
        if len(shape) not in (2, 3):
            raise ValueError("x must be [rows, cols] or [experts, rows, cols]")
        size = (shape[-2], shape[-1], shape[0] if len(shape) == 3 else 1)
        with _on(stream):
            out = Mx4(*size, data=torch.empty(Mx4.bytes_for(*size), dtype=torch.uint8, device=x.device))
    ld, le = _matrix(out, x, "x", dev)
    st = _lib.load().sg_mx4_quantize(out._c, kind, x.data_ptr(), ld, le, _s(stream, x))
    if st:
        _lib.check(st, "mx4_quantize")
    return out


def mx4_dequantize(m, out=None, dtype=torch.float32, stream=None):
    """The values of m, [rows, cols] ([experts, rows, cols] if it has several) of
    dtype, or into out."""
    if out is None:
        with _on(stream):
            out = torch.empty(*((m.experts,) if m.experts > 1 else ()), m.rows, m.cols, dtype=dtype, device=m.data.device)
    ld, le = _matrix(m, out, "out", _dev(out, "out"))
    st = _lib.load().sg_mx4_dequantize(m._c, _type(out, "out"), out.data_ptr(), ld, le, _s(stream, out))
    if st:
        _lib.check(st, "mx4_dequantize")
    return out


def _scratch_bytes(w, rows, desc):
    return _lib.load().sg_mx4_scratch_bytes(w._c, rows, desc)


def mx4_scratch(w, rows, stream=None):
    """Scratch of mx4_matmul for up to that many rows, or of mx4_experts for a MoePlan
    (rows), whatever it holds, up to its max_tokens: kept by the caller, one for calls
    that may overlap on the GPU."""
    if isinstance(rows, MoePlan):
        n = _scratch_bytes(w, 0, C.byref(SgMoePlan(rows.max_tokens, rows.n_used, rows.n_expert)))
    else:
        n = _scratch_bytes(w, rows, None)
    with _on(stream):
        return torch.empty(n, dtype=torch.uint8, device=w.data.device)


def _product(x, shape, w, up, out, dtype, rows, scratch, plan, stream):
    """What the two products have in common: the arguments of the call from x on (plan: an expert's, or None)."""
    dev, stride = _dev(x, "x"), x.stride()
    if len(shape) != 2 or shape[1] != w.cols or (stride[1] != 1 and shape[0]) or dev != w.dev:
        raise ValueError("x must be a tensor [rows, %d] with contiguous rows on the matrix's CUDA device" % w.cols)
    if up is not None and (up.experts != w.experts or up.rows != w.rows or up.cols != w.cols or up.dev != dev):
        raise ValueError("up must be a matrix of w's shape on the same CUDA device")
    if out is None:
        with _on(stream):
            out = torch.empty(rows, w.rows, dtype=dtype or x.dtype, device=x.device)
    n, feats = out.shape
    so = out.stride()
    if (n != rows or feats != w.rows or (so[1] != 1 and feats > 1 and rows) or out.get_device() != dev or
            (dtype is not None and dtype is not out.dtype)):
        raise ValueError("out must be a tensor [%d, %d] with contiguous rows on x's device" % (rows, w.rows))
    if scratch is None:
        with _on(stream):  # (of a plan, for the tokens that it holds)
            scratch = torch.empty(_scratch_bytes(w, rows, None) if plan is None else _scratch_bytes(w, 0, plan._c), dtype=torch.uint8, device=x.device)
    elif scratch.dtype is not torch.uint8 or not scratch.is_contiguous() or scratch.get_device() != dev:
        raise ValueError("scratch must be a contiguous uint8 tensor on x's device")
    return out, (_type(x, "x"), x.data_ptr(), stride[0]), (_type(out, "out"), out.data_ptr(), so[0], scratch.data_ptr(), scratch.numel(), _s(stream, x))


def mx4_matmul(x, w, up=None, out=None, dtype=None, scratch=None, stream=None):
    """x w^T for x [rows, w.cols] (float32, float16 or bfloat16), its rows quantized as
    w is, whatever their number; with up silu(x w^T) * (x up^T).  Returns out
    [rows, w.rows] of dtype (x's if None)."""
    shape = x.shape
    rows = shape[0]
    out, xs, rest = _product(x, shape, w, up, out, dtype, rows, scratch, None, stream)
    st = _lib.load().sg_mx4_matmul(w._c, None if up is None else up._c, *xs, rows, *rest)
    if st:
        _lib.check(st, "mx4_matmul")
    return out


class MoePlan:
    """Up to max_tokens tokens sorted by expert, n_used of n_expert each.  After
    moe_route or moe_sort of n tokens: ids and weights [n, n_used], first [n_expert +
    1], order [n * n_used] and place [n, n_used] (sg_moe_plan); they are the plan's and
    stay as they are until the next of these calls."""

    def __init__(self, max_tokens, n_used, n_expert, device="cuda"):
        i = lambda n: torch.empty(n, dtype=torch.int32, device=device)  # noqa: E731
        self.max_tokens, self.n_used, self.n_expert = max_tokens, n_used, n_expert
        work = _lib.load().sg_moe_plan_work_bytes(max_tokens, n_expert)
        if not work or not 0 < n_used <= _lib.MOE_MAX_USED or max_tokens * n_used >= 1 << 31:
            raise _lib.SgError(3, "moe_plan")
        n = max_tokens * n_used
        self._ids, self._order, self._place = i(n), i(n), i(n)
        self._weights = torch.empty(n, dtype=torch.float32, device=device)
        self.first, self._work = torch.zeros(n_expert + 1, dtype=torch.int32, device=device), torch.zeros(work // 4, dtype=torch.int32, device=device)
        self.dev = self.first.get_device()
        if self.dev < 0:
            raise ValueError("a plan must be CUDA memory")
        self.desc = SgMoePlan(0, n_used, n_expert, self._ids.data_ptr(), self._weights.data_ptr(), self.first.data_ptr(), self._order.data_ptr(),
                              self._place.data_ptr(), self._work.data_ptr())
        self._c = C.byref(self.desc)
        self._tokens(0)

    def _tokens(self, n):
        k = self.n_used
        self.n_tok = self.desc.n_tok = n
        self.ids, self.weights, self.place = (t[:n * k].view(n, k) for t in (self._ids, self._weights, self._place))
        self.order = self._order[:n * k]


def _plan(plan, n, t):
    if n > plan.max_tokens:
        raise ValueError("the plan is made for %d tokens" % plan.max_tokens)
    if plan.dev != _dev(t, "the tokens' tensor"):
        raise ValueError("the plan must lie on the same CUDA device")


def moe_route(logits, plan, norm=True, prune=0.0, stream=None):
    """The plan.n_used experts of each token by its logits [n, n_expert] (float32,
    float16 or bfloat16; minus infinity: not that one), their softmax weights (norm:
    over the chosen ones, otherwise over all) and the pairs sorted by expert
    (sg_moe_route).  prune as Moe's moe_prune.  Fills and returns plan."""
    shape, stride = logits.shape, logits.stride()
    if len(shape) != 2 or shape[1] != plan.n_expert or (stride[1] != 1 and shape[1] > 1):
        raise ValueError("logits must be a tensor [n, %d] with contiguous rows" % plan.n_expert)
    kind, n, was = _type(logits, "logits"), shape[0], plan.n_tok
    _plan(plan, n, logits)
    args = kind, logits.data_ptr(), stride[0], int(bool(norm)), float(prune), plan._c, _s(stream, logits)
    if was != n:
        plan._tokens(n)
    st = _lib.load().sg_moe_route(*args)
    if st:
        # the arrays on the device and the number of tokens belong together (the products take tiles and rows from the ones, the
        # sizes of what they read and write from the other): of a call that is refused they stay as they are, one that fails on
        # the way leaves no tokens
        plan._tokens(0 if st == _lib.ERR_CUDA else was)
        _lib.check(st, "moe_route")
    return plan


def moe_sort(ids, weights, plan, stream=None):
    """The pairs sorted by expert for choices of the caller's own: ids int32 and weights
    float32 [n, n_used] (ids outside the experts: none).  Fills and returns plan."""
    n = ids.shape[0]
    if ids.shape != (n, plan.n_used) or weights.shape != ids.shape or weights.dtype is not torch.float32 or weights.get_device() != plan.dev:
        raise ValueError("ids and weights must be int32 and float32 tensors [n, %d] of one CUDA device" % plan.n_used)
    _plan(plan, n, ids)
    _i32(ids, "ids", plan.dev)
    handle = _s(stream, ids)
    if plan.n_tok != n:
        plan._tokens(n)
    st = _lib.ERR_CUDA
    try:
        with _on(stream):
            for t, to in ((ids, plan.ids), (weights, plan.weights)):
                if n and not (t.data_ptr() == to.data_ptr() and t.is_contiguous()):  # (rows of the plan's own array: by way of others)
                    to.copy_(t.clone() if t.untyped_storage().data_ptr() == to.untyped_storage().data_ptr() else t)
        st = _lib.load().sg_moe_sort(plan._c, handle)
    finally:
        if st:  # (the ids have been written, or some of them)
            plan._tokens(0)
    if st:
        _lib.check(st, "moe_sort")
    return plan


def mx4_experts(x, w, plan, up=None, gather=None, out=None, dtype=None, scratch=None, stream=None):
    """The products of the plan's tokens with their experts (sg_mx4_experts): row s of
    the result, [n * n_used, w.rows] of dtype (x's if None), is that of sorted place s;
    with up silu(x w^T) * (x up^T).  x has a row per token (gather; the default where up
    is given) or per sorted place.  Rows past plan.first[-1] are left as they were."""
    gather = up is not None if gather is None else gather
    rows, shape = plan.n_tok * plan.n_used, x.shape
    if w.experts != plan.n_expert:
        raise ValueError("the plan has %d experts, the matrix %d" % (plan.n_expert, w.experts))
    if shape[0] != (plan.n_tok if gather else rows):
        raise ValueError("x must have a row per %s" % ("token" if gather else "sorted place"))
    if plan.dev != w.dev:
        raise ValueError("the plan must lie on the same CUDA device")
    out, xs, rest = _product(x, shape, w, up, out, dtype, rows, scratch, plan, stream)
    st = _lib.load().sg_mx4_experts(w._c, None if up is None else up._c, plan._c, *xs, 1 if gather else 0, *rest)
    if st:
        _lib.check(st, "mx4_experts")
    return out


def moe_combine(y, plan, out=None, dtype=None, stream=None):
    """The weighted sums of the experts' results (sg_moe_combine): y [n * n_used, dim],
    a row per sorted place, to out [n, dim] of dtype (y's if None)."""
    dev, shape, stride = _dev(y, "y"), y.shape, y.stride()
    if len(shape) != 2 or shape[0] != plan.n_tok * plan.n_used or (stride[1] != 1 and shape[1] > 1) or plan.dev != dev:
        raise ValueError("y must be a tensor [%d, dim] with contiguous rows on the plan's CUDA device" % (plan.n_tok * plan.n_used))
    dim = shape[1]
    if out is None:
        with _on(stream):
            out = torch.empty(plan.n_tok, dim, dtype=dtype or y.dtype, device=y.device)
    n, cols = out.shape
    so = out.stride()
    if (n != plan.n_tok or cols != dim or (so[1] != 1 and dim > 1) or out.get_device() != dev or
            (dtype is not None and dtype is not out.dtype)):
        raise ValueError("out must be a tensor [%d, %d] with contiguous rows on y's device" % (plan.n_tok, dim))
    st = _lib.load().sg_moe_combine(plan._c, _type(y, "y"), y.data_ptr(), stride[0], dim, _type(out, "out"), out.data_ptr(), so[0], _s(stream, y))
    if st:
        _lib.check(st, "moe_combine")
    return out
