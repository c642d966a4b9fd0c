"""CPU checks of what the Python entry points of the paged cache refuse: tensors of
the host, or of a GPU that is not the current one (a fake here)."""
import pytest
import torch

from spindle_b200 import kv4


class OnGpu(torch.Tensor):
    """A tensor that says it lies on a GPU."""
    where = 0

    def get_device(self):
        return self.where


def on(where, *n, dtype=torch.float32):
    t = torch.zeros(*n, dtype=dtype).as_subclass(OnGpu)
    t.where = where
    return t


def test_host_tensors():
    with pytest.raises(ValueError):
        kv4.logprobs(torch.zeros(2, 10))
    with pytest.raises(ValueError):
        kv4._dev(torch.zeros(2), "x")
    with pytest.raises(TypeError):
        kv4._i32(torch.zeros(2, dtype=torch.int32), "x", 0)
    with pytest.raises(ValueError):
        kv4._tables(torch.zeros(2, 2, dtype=torch.int32), 2, 0)


def test_a_gpu_that_is_not_the_current_one(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    assert kv4._dev(on(0, 3), "x") == 0
    with pytest.raises(ValueError):
        kv4._dev(on(1, 3), "x")
    with pytest.raises(ValueError):
        kv4.logprobs(on(1, 2, 10))
    with pytest.raises(TypeError):
        kv4._i32(on(1, 3, dtype=torch.int32), "x", 0)
    with pytest.raises(ValueError):
        kv4._tables(on(1, 2, 2, dtype=torch.int32), 2, 0)


def test_plan_refuses_overlapping_memory():
    # what a plan writes must not lie where it reads (addresses only: refused before a launch)
    import ctypes as C

    from spindle_b200 import _lib
    L = _lib.load()
    p = lambda k: C.c_void_p(0x100000 + k)  # noqa: E731
    at = dict(ctx=0x1000, new=0x2000, tables=0x3000, ring=0x4000, cursor=0x5000, cu=0x6000, seq=0x7000, pos=0x8000, slots=0x9000, info=0xa000)

    def plan(**kw):
        a = {k: p(v) for k, v in dict(at, **kw).items()}
        return L.sg_kv4_plan(64, 8, 10, a["ctx"], a["new"], a["tables"], 4, 4, a["ring"], a["cursor"], a["cu"], a["seq"], a["pos"],
                             a["slots"], 10, a["info"], None)
    sizes = dict(cu=44, seq=40, pos=40, slots=40, info=16, ring=32, tables=160)
    for read, n in (("ctx", 40), ("new", 40), ("cursor", 8)):
        for out, m in sizes.items():
            assert plan(**{out: at[read] + n - 4}) == 1, (read, out)
            assert plan(**{out: at[read] - m + 4}) == 1, (read, out)


def test_attention_refuses_tables_to_the_end_of_31_bits():
    # a step that begins below 2^31 may end past it
    import ctypes as C

    from spindle_b200 import _lib
    L = _lib.load()
    for page in (16, 64, 1024):
        cache = _lib.SgKv4(128, 8, page, 4, 0x100000)
        for past in (0, 16, 1024 - page):
            if past % page:
                continue
            a = _lib.SgKv4Attn(1, 8, 1, 1, 0x100000, 1024, 128, 0x100000, 1024, 128, None, 0x100000, 0x100000, 0x100000, 1 << 28,
                               ((1 << 31) - past) // page, 0.0, 0, 0, 0x100000, 1 << 30)
            assert L.sg_kv4_attention(C.byref(cache), C.byref(a), None) == 1, (page, past)
