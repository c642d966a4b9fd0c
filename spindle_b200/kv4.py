"""Paged KV cache held in 4 bits, for serving many requests: block tables and
slot maps from request lengths (kv4_plan), rows quantized into the cache
(kv4_append) and read back (kv4_read), grouped-query attention over it
(kv4_attention), and token log probabilities (logprobs), through the C ABI
(sg_kv4_*, sg_logprobs).  The reference keeps one f16 cache per chat
(smollm_chat.rs:2924-2972); nothing here changes that path (Decoder).

One serving step: plan, then per layer append and attend, then the LM head and
logprobs.  All lengths, tables and slots stay on the device."""
import contextlib
import ctypes as C

import torch

from . import _lib
from ._lib import SgKv4, SgKv4Attn

LOGPROBS_TOP_MAX = 64
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


def _s(stream, t):
    """The handle of the stream that a call on t's device runs on."""
    return torch._C._cuda_getCurrentRawStream(t.get_device()) if stream is None else stream.cuda_stream


def _on(stream):
    """What a call allocates belongs to the stream that it runs on."""
    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


def _type(t, what):
    try:
        return _TYPES[t.dtype]
    except KeyError:
        raise TypeError("%s must be float32, float16 or bfloat16" % what) from None


def _dev(t, what):
    """The index of t's GPU, which has to be the current one: the kernels run there, and
    every tensor of a call has to lie there."""
    d = t.get_device()
    if d < 0 or d != torch._C._cuda_getDevice():
        raise ValueError("%s must be a tensor of the current CUDA device" % what)
    return d


def _i32(t, what, dev, n=None):
    if t.dtype is not torch.int32 or t.get_device() != dev or not t.is_contiguous():
        raise TypeError("%s must be a contiguous int32 tensor of the same CUDA device" % what)
    if n is not None and t.numel() != n:
        raise ValueError("%s must have %d entries" % (what, n))
    return t.data_ptr()


def _tables(t, n, dev):
    """Pointer, row stride and width of a block table for n requests."""
    if t.dtype is not torch.int32 or t.dim() != 2 or t.get_device() != dev:
        raise ValueError("tables must be an int32 tensor [n_req, width] of the same CUDA device")
    rows, width = t.shape
    ld, one = t.stride()
    if rows != n or (one != 1 and width > 1 and rows):
        raise ValueError("tables must be int32 [%d, width] with contiguous rows" % n)
    return t.data_ptr(), ld, width


class Kv4Cache:
    """n_blocks blocks of `page` positions of n_kv_heads x head_dim K and V
    values in 4 bits (one per layer; 20 bytes per 32 values).  data:
    the device bytes (a uint8 CUDA tensor of Kv4Cache.bytes_for), allocated if None.
    nonfinite counts the groups of 32 appended values that had an infinity or a NaN."""

    def __init__(self, n_blocks, n_kv_heads, head_dim, page=64, device=None, data=None):
        self.n_blocks, self.n_kv_heads, self.head_dim, self.page = n_blocks, n_kv_heads, head_dim, page
        need = self.bytes_for(n_blocks, n_kv_heads, head_dim, page)
        if data is None:
            data = torch.zeros(need, dtype=torch.uint8, device=device or "cuda")
        if data.dtype != torch.uint8 or not data.is_cuda or not data.is_contiguous() or data.numel() < need:
            raise ValueError("data must be a contiguous uint8 CUDA tensor of %d bytes" % need)
        self.data, self.dev = data, data.get_device()
        self.nonfinite = torch.zeros(1, dtype=torch.int32, device=data.device)
        self._nonfinite = self.nonfinite.data_ptr()
        self.desc = SgKv4(head_dim, n_kv_heads, page, n_blocks, data.data_ptr())
        self._c = C.byref(self.desc)

    @staticmethod
    def bytes_for(n_blocks, n_kv_heads, head_dim, page):
        n = _lib.load().sg_kv4_bytes(C.byref(SgKv4(head_dim, n_kv_heads, page, n_blocks, None)))
        if not n:
            raise _lib.SgError(3, "kv4_bytes")
        return n


class Kv4Plan:
    """What kv4_plan writes, for up to n_req requests and max_tokens new
    positions a step: cu [n_req + 1], seq [n_req], pos and slots [max_tokens],
    and info [4] (the next step's cursor, the sum of the new positions, the
    blocks that were wanted and not there; of the last call).  It also keeps a ring
    of all blocks, free to begin with, and the cursor, for callers without their own."""

    def __init__(self, n_req, max_tokens, page, n_blocks, device="cuda"):
        new = lambda n: torch.empty(n, dtype=torch.int32, device=device)  # noqa: E731
        self.n_req, self.max_tokens, self.page, self.n_blocks = n_req, max_tokens, page, n_blocks
        self.cu, self.seq, self.pos, self.slots = new(n_req + 1), new(n_req), new(max_tokens), new(max_tokens)
        self.ring = torch.arange(n_blocks, dtype=torch.int32, device=device)
        # two a kind, as a call reads a cursor and writes the next: of the own ring, and of rings that are given
        infos = torch.tensor([[0, n_blocks, 0, 0]] * 4, dtype=torch.int32, device=device).unbind()
        self._infos, self._given = infos[:2], infos[2:]
        self._turn = self._given_turn = 0
        self._captured = False  # a graph holds the own ring's cursor: it stays where it is
        self.info = self._infos[0]
        self.dev = self.ring.get_device()
        self._out = (self.cu.data_ptr(), self.seq.data_ptr(), self.pos.data_ptr(), self.slots.data_ptr())


def kv4_plan(plan, ctx, new, tables, ring=None, cursor=None, stream=None):
    """Block tables and slot maps of one step (sg_kv4_plan): ctx and new int32
    [n_req] (positions held, positions to come; new < 0: the request ends; ctx may
    be plan.seq, to carry the lengths on in place), tables
    int32 [n_req, width], updated in place.  ring and cursor: the free blocks
    (int32 [n_blocks] and [2 or more]; info[:2] is the next call's cursor); None: the
    plan's own, carried from call to call, replays of captured calls among them.
    Fills and returns plan."""
    n = ctx.numel()
    if n != plan.n_req:
        raise ValueError("the plan is made for %d requests" % plan.n_req)
    dev = _dev(tables, "tables")
    if plan.dev != dev:
        raise ValueError("the plan must lie on the same CUDA device")
    table, ld, width = _tables(tables, n, dev)
    if (ring is None) != (cursor is None):
        raise ValueError("ring and cursor come together")
    own = cursor is None
    if own:
        turn = plan._turn ^ 1
        ring, cursor, info = plan.ring, plan._infos[plan._turn], plan._infos[turn]
    elif ring.numel() != plan.n_blocks or cursor.numel() < 2:
        raise ValueError("ring must have n_blocks entries and cursor two")
    else:
        turn = plan._given_turn ^ 1
        if plan._given[turn].data_ptr() == cursor.data_ptr():
            turn ^= 1
        info = plan._given[turn]
    cu, seq, pos, slots = plan._out
    st = _lib.load().sg_kv4_plan(plan.page, plan.n_blocks, n, _i32(ctx, "ctx", dev), _i32(new, "new", dev, n), table,
                                 ld, width, _i32(ring, "ring", dev), _i32(cursor, "cursor", dev), cu, seq, pos,
                                 slots, plan.max_tokens, info.data_ptr(), _s(stream, tables))
    if st:
        _lib.check(st, "kv4_plan")
    if not own:
        plan._given_turn = turn
    else:
        with _on(stream):
            if plan._captured or torch.cuda.is_current_stream_capturing():
                # a replay reads the cursor where the captured call did: the next one goes there, from now on for
                # the calls outside the graph too
                cursor = plan._infos[plan._turn]
                cursor.copy_(info)
                plan._captured, info = True, cursor
            else:
                plan._turn = turn
    plan.info = info
    return plan


def _rows(cache, t, what):
    """Number, token and head stride of rows of the cache's heads."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[1] != cache.n_kv_heads or shape[2] != cache.head_dim or stride[2] != 1 or t.get_device() != cache.dev:
        raise ValueError("%s must be a tensor [n_tok, %d, %d] with contiguous rows on the cache's CUDA device" %
                         (what, cache.n_kv_heads, cache.head_dim))
    return shape[0], stride[0], stride[1]


def kv4_append(cache, k, v, slots, stream=None):
    """Quantizes the rows k, v [n_tok, n_kv_heads, head_dim] (float32, float16 or
    bfloat16, any token and head strides) into their slots (int32 [n_tok], as
    kv4_plan makes them; negative: the row is left out)."""
    dev = _dev(k, "k")
    n, kt, kh = _rows(cache, k, "k")
    nv, vt, vh = _rows(cache, v, "v")
    if v.dtype is not k.dtype or nv != n:
        raise ValueError("k and v must have one type and one number of rows")
    st = _lib.load().sg_kv4_append(cache._c, _type(k, "k"), k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, _i32(slots, "slots", dev, n), n,
                                   cache._nonfinite, _s(stream, k))
    if st:
        _lib.check(st, "kv4_append")


def kv4_read(cache, slots, out=None, dtype=torch.float16, stream=None):
    """The values that the cache holds at the given slots (int32 [n_tok]): (k, v),
    [n_tok, n_kv_heads, head_dim] of dtype each, or into out = (k, v)."""
    n, dev = slots.numel(), _dev(slots, "slots")
    if out is None:
        with _on(stream):
            out = tuple(torch.empty(n, cache.n_kv_heads, cache.head_dim, dtype=dtype, device=slots.device)
                        for _ in range(2))
    k, v = out
    if (_rows(cache, k, "out")[0] != n or _rows(cache, v, "out")[0] != n or v.dtype is not k.dtype or not k.is_contiguous() or
            not v.is_contiguous()):
        raise ValueError("out must be two contiguous tensors of one type with a row per slot")
    st = _lib.load().sg_kv4_read(cache._c, _type(k, "out"), _i32(slots, "slots", dev), n, k.data_ptr(), v.data_ptr(), _s(stream, k))
    if st:
        _lib.check(st, "kv4_read")
    return out


def kv4_attention_scratch(device="cuda", stream=None):
    """Scratch of kv4_attention: kept by the caller, one for calls that may overlap on the GPU."""
    L = _lib.load()
    with _on(stream):
        t = torch.empty(L.sg_kv4_attention_scratch_bytes(), dtype=torch.uint8, device=device)
    if not t.is_cuda:
        raise ValueError("scratch must be CUDA memory")
    _lib.check(L.sg_kv4_attention_scratch_init(t.data_ptr(), t.numel(), _s(stream, t)), "kv4_attention_scratch_init")
    return t


def kv4_attention(cache, q, cu, seq, tables, scale=None, window=0, max_new=0, out=None, lse=None, scratch=None, stream=None):
    """Grouped-query attention of new tokens over the cache (sg_kv4_attention): q
    [n_tok, n_heads, head_dim] (float32, float16 or bfloat16), cu [n_req + 1] and
    seq [n_req] int32 as kv4_plan makes them, tables int32 [n_req, width].  Token t
    of a request sees the positions up to its own, the last `window` of them if
    window > 0.  scale None: 1 / sqrt(head_dim) (0: equal weights).  max_new: an upper bound of a request's new tokens, if the caller
    knows one (tokens past one that is too small may get NaN).  lse: optional float32 [n_tok, n_heads] to fill with the log of the
    softmax's sum.  Returns out, [n_tok, n_heads, head_dim] of q's type."""
    n = seq.numel()
    shape, stride = q.shape, q.stride()
    dev = _dev(q, "q")
    if len(shape) != 3 or shape[2] != cache.head_dim or stride[2] != 1 or dev != cache.dev:
        raise ValueError("q must be a tensor [n_tok, n_heads, %d] with contiguous rows on the cache's CUDA device" % cache.head_dim)
    table, ld, width = _tables(tables, n, dev)
    if out is None:
        with _on(stream):
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
    ostride = out.stride()
    if out.shape != shape or out.dtype is not q.dtype or ostride[2] != 1 or out.get_device() != dev:
        raise ValueError("out must have q's shape, type and device, and contiguous rows")
    if lse is not None and (lse.dtype is not torch.float32 or lse.shape != shape[:2] or not lse.is_contiguous() or lse.get_device() != dev):
        raise ValueError("lse must be a contiguous float32 [n_tok, n_heads] on q's device")
    if scratch is None:
        scratch = kv4_attention_scratch(q.device, stream)
    elif not scratch.is_contiguous() or scratch.get_device() != dev:
        raise ValueError("scratch must be a contiguous tensor on q's device")
    a = SgKv4Attn(_type(q, "q"), shape[1], shape[0], n, q.data_ptr(), stride[0], stride[1], out.data_ptr(), ostride[0], ostride[1],
                  None if lse is None else lse.data_ptr(), _i32(cu, "cu", dev, n + 1), _i32(seq, "seq", dev), table, ld, width,
                  0.0 if scale is None else 1e-38 if -1e-38 < scale < 1e-38 else scale, window, max_new, scratch.data_ptr(), scratch.numel())
    st = _lib.load().sg_kv4_attention(cache._c, C.byref(a), _s(stream, q))
    if st:
        _lib.check(st, "kv4_attention")
    return out


class LogProbs:
    """What logprobs returns, for `rows` rows: logprob and entropy float32 [rows],
    rank int32 [rows], top_ids int32 and top_logprobs float32 [rows, top]."""

    def __init__(self, rows, top=0, device="cuda"):
        f = lambda *n: torch.empty(*n, dtype=torch.float32, device=device)  # noqa: E731
        i = lambda *n: torch.empty(*n, dtype=torch.int32, device=device)  # noqa: E731
        self.rows, self.top = rows, top
        self.logprob, self.entropy, self.rank = f(rows), f(rows), i(rows)
        self.top_ids, self.top_logprobs = i(rows, top), f(rows, top)
        self.dev = self.rank.get_device()
        self._p = [t.data_ptr() for t in (self.logprob, self.entropy, self.rank, self.top_ids, self.top_logprobs)]


def logprobs(logits, tokens=None, top=0, out=None, stream=None):
    """Log probabilities of the given tokens under softmax(logits) (sg_logprobs):
    logits [rows, vocab] float32, float16 or bfloat16 with contiguous rows, tokens
    int32 [rows] or None, top up to 64 alternatives.  Returns a LogProbs (out, if
    given): the log probability and the rank (0: the likeliest) of each given
    token, the entropy in nats, and the `top` likeliest tokens."""
    shape, stride = logits.shape, logits.stride()
    dev = _dev(logits, "logits")
    if len(shape) != 2 or (stride[1] != 1 and shape[1] > 1):
        raise ValueError("logits must be a tensor [rows, vocab] with contiguous rows")
    rows, vocab = shape
    if out is None:
        with _on(stream):
            out = LogProbs(rows, top, logits.device)
    elif out.rows != rows or out.top != top:
        raise ValueError("out is made for %d rows and top %d" % (out.rows, out.top))
    elif out.dev != dev:
        raise ValueError("out must lie on the logits' device")
    lp, ent, rank, ids, tops = out._p
    st = _lib.load().sg_logprobs(_type(logits, "logits"), logits.data_ptr(), stride[0], rows, vocab,
                                 None if tokens is None else _i32(tokens, "tokens", dev, rows), lp, ent, rank, top, ids, tops,
                                 _s(stream, logits))
    if st:
        _lib.check(st, "logprobs")
    return out
