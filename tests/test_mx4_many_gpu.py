"""The kernel for many tokens on the GPU: every tile width, type and alignment of its results,
columns of one stage and of more than its ring has, part-filled tiles, and several tiles a pair
of SMs in turn."""
import ctypes as C

import pytest
import torch

import mx4_util as U
import spindle_b200 as sg
from spindle_b200 import _lib

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rand(dev, *shape, seed=0):
    return torch.randn(*shape, device=dev, generator=torch.Generator(device=dev).manual_seed(seed))


def same_in_all_types(x):
    """Values that f16 and bf16 hold too, up to 8 in steps of 1/16."""
    return (x.clamp(-7.9, 7.9) * 16).round() / 16


def tile(w, n, dual=False):
    """Which kernel a product of n rows (or of a plan) is run by, and its tokens a tile."""
    many, rows = C.c_int32(), C.c_int32()
    a = (0, n._c) if isinstance(n, sg.MoePlan) else (n, None)
    _lib.check(_lib.load().sg_mx4_tile(w._c, int(dual), *a, C.byref(many), C.byref(rows)), "mx4_tile")
    return many.value, rows.value


def check_places(call, want, bound, used, feats):
    """call(out) for results of all types, in rows that begin on 16 bytes, on 4, on 2 and between: within bound where they
    are, nothing written elsewhere."""
    rows = want.shape[0]
    for dtype in TYPES:
        for off, ld in ((0, feats + 24 - feats % 8), (2, feats + 4 + feats % 2), (1, feats + 3 + feats % 2)):
            out = torch.full((rows + 2, ld), 7.0, dtype=dtype, device=want.device)
            y = out[1:-1, off:off + feats]
            call(y)
            assert U.close(y[:used], want[:used], bound[:used])
            y[:used] = 7.0
            assert (out == 7).all()


# rows, columns, features, tokens a tile
@pytest.mark.parametrize("rows,cols,n,width", [(2600, 64, 1100, 192), (2600, 544, 1025, 192), (1281, 1824, 2050, 192), (5000, 320, 2000, 192),
                                               (1500, 2048, 3001, 256), (2305, 1440, 1300, 256), (5041, 544, 2599, 256)])
def test_matmul_of_many(dev, rows, cols, n, width):
    x, w = same_in_all_types(rand(dev, rows, cols, seed=rows)), rand(dev, n, cols, seed=n) * cols ** -0.5
    up = rand(dev, n, cols, seed=n + 1) * cols ** -0.5
    W, V = sg.mx4_quantize(w), sg.mx4_quantize(up)
    xq, wq, vq = U.quantized(x), U.quantized(w), U.quantized(up)
    assert tile(W, rows) == (1, width) and tile(W, rows, dual=True) == (1, 128)
    for v, q in ((None, None), (V, vq)):
        want, bound = U.product(xq, wq, q)
        check_places(lambda out: sg.mx4_matmul(x, W, up=v, out=out), want, bound, rows, n)  # noqa: B023
        for dtype in TYPES[1:]:
            assert U.close(sg.mx4_matmul(x.to(dtype), W, up=v, dtype=torch.float32), want, bound)
    assert torch.equal(sg.mx4_matmul(x, W, up=V), sg.mx4_matmul(x, W, up=V))
    sg.device_status()


# the columns on both sides of what takes tiles of 256 tokens; experts without tokens and crowded ones
@pytest.mark.parametrize("n,e,k,dim,ff,width", [(300, 40, 6, 544, 257, 192), (3000, 5, 2, 320, 300, 192), (1500, 12, 4, 2080, 384, 256),
                                                (700, 64, 8, 1856, 130, 256)])
@pytest.mark.parametrize("uneven", [0.5, 3.0])
def test_experts_of_many(dev, n, e, k, dim, ff, width, uneven):
    x = same_in_all_types(rand(dev, n, dim, seed=n))
    logits = rand(dev, n, e, seed=1) + uneven * rand(dev, e, seed=2)
    logits[:, 0] = logits[n // 2:, -1] = logits[0] = float("-inf")  # an expert and a token without any, one for some
    gate, up, down = rand(dev, e, ff, dim, seed=3) * dim ** -0.5, rand(dev, e, ff, dim, seed=4) * dim ** -0.5, rand(dev, e, dim, ff // 32 * 32, seed=5) * ff ** -0.5
    G, V, D = (sg.mx4_quantize(t) for t in (gate, up, down))
    p = sg.moe_route(logits, sg.MoePlan(n, k, e, device=dev))
    assert tile(G, p) == (1, width) and tile(G, p, dual=True) == (1, 128) and tile(D, p)[0] == 1
    first, used = p.first.tolist(), int(p.first[-1])
    assert used < n * k
    xq = U.quantized(x)[p.order[:used].long() // k]

    def one_by_one(rows, *ws):
        y = [U.product(rows[first[i]:first[i + 1]], *[q[i] for q in ws]) for i in range(e)]
        rest = torch.zeros(n * k - used, y[0][0].shape[1], dtype=torch.float64, device=dev)
        return [torch.cat([t[j] for t in y] + [rest]) for j in (0, 1)]
    gq, vq, dq = (U.quantized(t) for t in (gate, up, down))
    check_places(lambda out: sg.mx4_experts(x, G, p, up=V, out=out), *one_by_one(xq, gq, vq), used, ff)
    check_places(lambda out: sg.mx4_experts(x, G, p, gather=True, out=out), *one_by_one(xq, gq), used, ff)
    h = same_in_all_types(rand(dev, n * k, ff // 32 * 32, seed=6))
    h[used:] = float("nan")                                         # places that no pair has
    check_places(lambda out: sg.mx4_experts(h, D, p, out=out), *one_by_one(U.quantized(h[:used]), dq), used, dim)
    for dtype in TYPES[1:]:
        want, bound = one_by_one(U.quantized(h[:used]), dq)
        assert U.close(sg.mx4_experts(h.to(dtype), D, p, dtype=torch.float32)[:used], want[:used], bound[:used])
    sg.device_status()


@pytest.mark.parametrize("dual", [False, True])
def test_many_captured_and_on_two_streams(dev, dual):
    rows, cols, n = 1500, 320, 2100
    W, V = sg.mx4_quantize(rand(dev, n, cols, seed=1) * 0.06), sg.mx4_quantize(rand(dev, n, cols, seed=2) * 0.06)
    up = V if dual else None
    x = rand(dev, rows, cols, seed=3)
    assert tile(W, rows, dual=dual)[0] == 1
    scratch, out = sg.mx4_scratch(W, rows), torch.empty(rows, n, device=dev)
    sg.mx4_matmul(x, W, up=up, out=out, scratch=scratch)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sg.mx4_matmul(x, W, up=up, out=out, scratch=scratch)
    for seed in (4, 5):
        x.copy_(rand(dev, rows, cols, seed=seed))
        g.replay()
        assert torch.equal(out, sg.mx4_matmul(x, W, up=up))
    xs, side = [rand(dev, rows, cols, seed=6 + i) for i in range(2)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [sg.mx4_matmul(xs[i % 2], W, up=up, stream=side[i % 2]) for i in range(6)]
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, sg.mx4_matmul(xs[i % 2], W, up=up))
    sg.device_status()


@pytest.mark.parametrize("dual", [False, True])
def test_many_nonfinite_rows_stay_apart(dev, dual):
    rows, cols, n = 2100, 544, 1500
    x, w = rand(dev, rows, cols, seed=5), rand(dev, n, cols, seed=6)
    W = sg.mx4_quantize(torch.cat([w[:17], torch.full((1, cols), float("nan"), device=dev), w[18:]]))
    x[::3, 100], x[1::30, 300] = float("nan"), float("inf")
    y = sg.mx4_matmul(x, W, up=sg.mx4_quantize(w) if dual else None)
    assert tile(W, rows, dual)[0] == 1
    nan = torch.zeros(rows, n, dtype=torch.bool, device=dev)
    nan[::3] = nan[1::30] = True
    nan[:, 17] = True
    assert torch.equal(y.isnan(), nan)


# places of an expert on average up to 32 and from 33 on; experts of all numbers of tokens, tiles of 32 in part and several
@pytest.mark.parametrize("n,e,k,tile_of", [(256, 16, 2, (0, 32)), (264, 16, 2, (0, 128)), (16, 128, 2, (0, 32)), (1024, 64, 2, (0, 32)), (1056, 64, 2, (1, 192)),
                                           (32, 1, 1, (0, 32)), (33, 1, 1, (0, 128))])
@pytest.mark.parametrize("uneven", [0.0, 2.0])
def test_few_places_an_expert(dev, n, e, k, tile_of, uneven):
    dim, ff = 288, 200
    x, w = rand(dev, n, dim, seed=n), rand(dev, e, ff, dim, seed=3) * dim ** -0.5
    W = sg.mx4_quantize(w)
    p = sg.moe_route(rand(dev, n, e, seed=1) + uneven * rand(dev, e, seed=2), sg.MoePlan(n, k, e, device=dev))
    assert tile(W, p) == tile_of
    y, first, wq = sg.mx4_experts(x, W, p, gather=True), p.first.tolist(), U.quantized(w)
    xq = U.quantized(x)[p.order.long() // k]
    for i in range(e):
        assert U.close(y[first[i]:first[i + 1]], *U.product(xq[first[i]:first[i + 1]], wq[i]))
    sg.device_status()
