"""The paged 4-bit KV cache on the GPU at the edges of what its entry points take."""
import pytest
import torch

import kv4_util as U
import spindle_b200 as sg
from test_kv4_gpu import TYPES, case, check, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_tok,heads,group", [(1, 1, 1), (1, 2, 7), (3, 2, 2), (2000, 4, 8)])
def test_attention_without_requests(dev, dtype, n_tok, heads, group):
    # tokens that belong to no request, and no request at all
    cache = sg.Kv4Cache(2, heads, 64, 16, device=dev)
    q = torch.randn(n_tok, heads * group, 64, device=dev).to(dtype)
    lse = torch.zeros(n_tok, heads * group, device=dev)
    for width in (0, 3):
        out = sg.kv4_attention(cache, q, ints([0], dev), ints([], dev), torch.empty(0, width, dtype=torch.int32, device=dev), lse=lse)
        assert (out == 0).all() and torch.isneginf(lse).all()
    sg.device_status()


def test_tensors_of_another_device_are_refused(dev):
    # every argument that a kernel reads or writes: memory of the host is refused before a launch
    cpu = lambda *n, dtype=torch.float32: torch.zeros(*n, dtype=dtype)  # noqa: E731
    gpu = lambda *n, dtype=torch.float32: torch.zeros(*n, dtype=dtype, device=dev)  # noqa: E731
    i32 = torch.int32
    cache = sg.Kv4Cache(4, 2, 64, 16, device=dev)
    scratch = sg.kv4_attention_scratch(dev)
    good = dict(q=gpu(1, 4, 64), cu=ints([0, 1], dev), seq=ints([1], dev), tables=ints([[0]], dev), out=gpu(1, 4, 64), lse=gpu(1, 4),
                scratch=scratch)
    sg.kv4_attention(cache, **good)
    for name, t in good.items():
        with pytest.raises((ValueError, TypeError)):
            sg.kv4_attention(cache, **dict(good, **{name: t.cpu()}))
    with pytest.raises(ValueError):     # 16 MB by its count of entries only
        sg.kv4_attention(cache, **dict(good, scratch=scratch[:1].expand(scratch.numel())))
    with pytest.raises(ValueError):
        sg.kv4_attention_scratch("cpu")
    with pytest.raises(ValueError):
        sg.Kv4Cache(4, 2, 64, 16, data=cpu(1 << 20, dtype=torch.uint8))
    k, slots = gpu(1, 2, 64), ints([0], dev)
    for bad in ((k.cpu(), k, slots), (k, k.cpu(), slots), (k, k, slots.cpu())):
        with pytest.raises((ValueError, TypeError)):
            sg.kv4_append(cache, *bad)
    for bad in ((slots.cpu(), (k, k)), (slots, (k.cpu(), k)), (slots, (k, k.cpu()))):
        with pytest.raises((ValueError, TypeError)):
            sg.kv4_read(cache, bad[0], out=bad[1])
    z, t, ring, cursor = ints([0, 0], dev), ints([[0], [0]], dev), gpu(4, dtype=i32), ints([0, 4], dev)
    plan = sg.Kv4Plan(2, 4, 16, 4, device=dev)
    for bad in ((z.cpu(), z, t, ring, cursor), (z, z.cpu(), t, ring, cursor), (z, z, t.cpu(), ring, cursor), (z, z, t, ring.cpu(), cursor),
                (z, z, t, ring, cursor.cpu())):
        with pytest.raises((ValueError, TypeError)):
            sg.kv4_plan(plan, *bad)
    with pytest.raises(ValueError):
        sg.kv4_plan(sg.Kv4Plan(2, 4, 16, 4, device="cpu"), z, z, t)
    x, tok = gpu(2, 100), ints([1, 2], dev)
    for args, out in (((x.cpu(), tok), None), ((x, tok.cpu()), None), ((x, tok), sg.LogProbs(2, 0, device="cpu"))):
        with pytest.raises((ValueError, TypeError)):
            sg.logprobs(*args, out=out)
    torch.cuda.synchronize()


@pytest.mark.parametrize("heads,group,new", [(2, 4, 3), (2, 4, 300), (4, 8, 900)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_means_of_f16s_largest_number(dev, d, heads, group, new):
    # V equal to +-65504 in some groups: a mean of it is that number, whatever the weights' rounding (which shows most
    # where one position that comes late has nearly all the weight, hence the scale)
    page, length, scale = 16, 1000, 4 * d ** -0.5
    cache = sg.Kv4Cache(63, heads, d, page, device=dev)
    g = torch.Generator(device=dev).manual_seed(new)
    k, v = (torch.randn(length, heads, d, device=dev, generator=g) for _ in range(2))
    v[..., :32], v[..., 32:64] = 65504.0, -65504.0
    sg.kv4_append(cache, k, v, torch.arange(length, dtype=torch.int32, device=dev))
    tables = torch.arange(63, dtype=torch.int32, device=dev)[None]
    for dtype in TYPES:
        q = torch.randn(new, heads * group, d, device=dev, generator=g).to(dtype)
        out = sg.kv4_attention(cache, q, ints([0, new], dev), ints([length], dev), tables, scale=scale)
        check(dev, cache, tables, tables.cpu(), ints([0, new], dev), ints([length], dev), q, scale, 0, out, None)
