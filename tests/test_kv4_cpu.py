"""CPU checks of the paged 4-bit cache and log-probability entry points: sizes,
and bad arguments refused before anything is launched."""
import ctypes as C

from spindle_b200 import _lib

FAKE = C.c_void_p(0x100000)


def cache(d=128, heads=8, page=64, blocks=4, data=0x100000):
    return C.byref(_lib.SgKv4(d, heads, page, blocks, data))


def attn(**kw):
    f = dict(type=1, n_heads=8, n_tok=1, n_req=1, q=0x100000, q_tok=1024, q_head=128, out=0x100000, o_tok=1024, o_head=128,
             lse=None, cu=0x100000, seq=0x100000, tables=0x100000, ld_tables=4, width=4, scale=0.0, window=0, max_new=0,
             scratch=0x100000, scratch_bytes=1 << 30)
    f.update(kw)
    return C.byref(_lib.SgKv4Attn(**f))


def test_cache_bytes():
    L = _lib.load()
    for d in (64, 128, 256):
        assert L.sg_kv4_bytes(cache(d, 8, 64, 4)) == 4 * 8 * 64 * d * 2 * 5 // 8
    for bad in (cache(96), cache(page=8), cache(page=48), cache(page=2048), cache(heads=0), cache(blocks=0),
                cache(page=1024, blocks=1 << 21), None):
        assert L.sg_kv4_bytes(bad) == 0


def test_struct_sizes_match_the_header():
    # the C layout: no padding surprises between Python and the library
    assert C.sizeof(_lib.SgKv4) == 24
    assert C.sizeof(_lib.SgKv4Attn) == 152
    assert _lib.SgKv4Attn.scale.offset == 120 and _lib.SgKv4Attn.scratch_bytes.offset == 144


def test_attention_refusals():
    L = _lib.load()
    assert L.sg_kv4_attention(None, attn(), None) == 1
    assert L.sg_kv4_attention(cache(), None, None) == 1
    assert L.sg_kv4_attention(cache(d=80), attn(), None) == 3
    assert L.sg_kv4_attention(cache(data=None), attn(), None) == 1
    assert L.sg_kv4_attention(cache(data=0x100008), attn(), None) == 4
    assert L.sg_kv4_attention(cache(), attn(type=8), None) == 2
    for bad in (dict(q=None), dict(out=None), dict(cu=None), dict(seq=None), dict(tables=None), dict(scratch=None),
                dict(scratch_bytes=100), dict(scale=float("inf")), dict(scale=float("nan")), dict(width=1 << 26),
                dict(n_tok=1 << 31), dict(n_req=1 << 31), dict(n_req=2, ld_tables=3)):
        assert L.sg_kv4_attention(cache(), attn(**bad), None) == 1, bad
    assert L.sg_kv4_attention(cache(), attn(n_heads=12), None) == 3
    assert L.sg_kv4_attention(cache(), attn(n_heads=0), None) == 3
    assert L.sg_kv4_attention(cache(), attn(q=0x100001), None) == 4
    assert L.sg_kv4_attention(cache(), attn(scratch=0x100010), None) == 4
    assert L.sg_kv4_attention(cache(), attn(n_tok=0), None) == 0  # nothing to do
    assert L.sg_kv4_attention_scratch_init(FAKE, 16, None) == 1


def test_append_read_plan_and_logprobs_refusals():
    L = _lib.load()
    app = lambda c, ty, k, v, s, n: L.sg_kv4_append(c, ty, k, 1024, 128, v, 1024, 128, s, n, None, None)  # noqa: E731
    assert app(cache(), 12, FAKE, FAKE, FAKE, 1) == 2
    assert app(cache(), 1, None, FAKE, FAKE, 1) == 1
    assert app(cache(), 1, FAKE, FAKE, None, 1) == 1
    assert app(cache(), 0, C.c_void_p(0x100002), FAKE, FAKE, 1) == 4
    assert app(cache(d=32), 0, FAKE, FAKE, FAKE, 1) == 3
    assert app(cache(), 1, None, None, None, 0) == 0
    assert L.sg_kv4_read(cache(), 1, FAKE, 1, None, FAKE, None) == 1
    assert L.sg_kv4_read(cache(), 1, FAKE, 1, C.c_void_p(0x100008), FAKE, None) == 4
    assert L.sg_kv4_read(cache(), 9, FAKE, 1, FAKE, FAKE, None) == 2

    def plan(page=64, blocks=8, n=2, ctx=FAKE, ring=FAKE, cursor=C.c_void_p(0x200000), info=FAKE, ld=4, width=4, pos=FAKE):
        return L.sg_kv4_plan(page, blocks, n, ctx, FAKE, FAKE, ld, width, ring, cursor, FAKE, FAKE, pos, FAKE, 10, info, None)
    assert plan(page=17) == 3
    assert plan(blocks=0) == 3
    assert plan(ctx=None) == 1
    assert plan(ring=None) == 1
    assert plan(cursor=FAKE) == 1      # the same memory as info
    assert plan(ld=3) == 1
    assert plan(pos=None) == 1
    assert plan(n=1 << 31) == 1

    def lp(ty=0, x=FAKE, ld=100, rows=2, vocab=100, top=0, ids=None):
        return L.sg_logprobs(ty, x, ld, rows, vocab, None, FAKE, FAKE, FAKE, top, ids, ids, None)
    assert lp(ty=14) == 2
    assert lp(x=None) == 1
    assert lp(x=C.c_void_p(0x100002)) == 4
    assert lp(vocab=0) == 3
    assert lp(vocab=(1 << 30) + 1) == 3
    assert lp(top=65, ids=FAKE) == 3
    assert lp(top=5) == 1
    assert lp(ld=99) == 1
    assert lp(rows=0) == 0
