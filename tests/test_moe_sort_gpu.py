"""Tokens sorted by expert on the GPU: the choice, the sort, the experts' products and
the weighted sum back."""
import pytest
import torch

import mx4_util as U
import spindle_b200 as sg

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rand(dev, *shape, seed=0):
    return torch.randn(*shape, device=dev, generator=torch.Generator(device=dev).manual_seed(seed))


def check_sort(p, ids, n_expert):
    for got, want in zip((p.first, p.order, p.place), U.sort(ids.cpu(), n_expert)):
        assert torch.equal(got.cpu(), want)


# (softmax weights: exponential, sum and quotient in f32, a few half steps each: 40 of them, 2.4e-6)
@pytest.mark.parametrize("n,e,k", [(1, 1, 1), (1, 128, 8), (3, 5, 4), (16, 128, 8), (63, 60, 6), (64, 256, 16), (65, 257, 2), (200, 1000, 16), (777, 1024, 3),
                                   (129, 8, 8), (500, 512, 5)])
@pytest.mark.parametrize("norm", [True, False])
def test_route(dev, n, e, k, norm):
    for dtype in TYPES:
        x = (rand(dev, n, e, seed=n + e) * 2).to(dtype)   # (16-bit logits have ties)
        x[rand(dev, n, e, seed=9) > 1.0] = float("-inf")
        p = sg.moe_route(x, sg.MoePlan(n + 7, k, e, device=dev), norm=norm)
        ids, w = U.choice(x, k, norm)
        assert torch.equal(p.ids.cpu(), ids)
        assert ((p.weights.double().cpu() - w).abs() <= 2.4e-6 * w).all()
        check_sort(p, ids, e)


@pytest.mark.parametrize("prune", [0.05, 0.3, 0.9, 1.0, 3.0, 100.0])
def test_route_prunes(dev, prune):
    x = rand(dev, 300, 64, seed=3) * 2
    x[5] = float("-inf")
    x[6, 2:] = float("-inf")
    for k in (1, 2, 3, 8):
        p = sg.moe_route(x, sg.MoePlan(300, k, 64, device=dev), prune=prune)
        ids, w = U.choice(x, k, True, prune)
        assert torch.equal(p.ids.cpu(), ids) and ((p.weights.double().cpu() - w).abs() <= 2.4e-6 * w).all()
        check_sort(p, ids, 64)


def test_route_edges(dev):
    x = torch.zeros(8, 40, device=dev)
    x[1] = float("-inf")                          # no expert is left
    x[2, 3] = float("inf")
    x[3, 7] = float("nan")
    x[4] = -0.0
    x[4, 9] = 0.0                                 # equal to the others
    x[5] = torch.finfo(torch.float32).min         # a mask of the lowest value is a value
    x[6, :38] = float("-inf")
    p = sg.moe_route(x, sg.MoePlan(8, 4, 40, device=dev))
    ids, w = p.ids.cpu(), p.weights.cpu()
    assert ids[0].tolist() == [0, 1, 2, 3] and (w[0] == 0.25).all()
    assert ids[1].tolist() == [-1] * 4 and (w[1] == 0).all()
    assert ids[2].tolist() == [3, 0, 1, 2] and w[2, 0].isnan()
    assert ids[3].tolist() == [7, 0, 1, 2] and w[3].isnan().all()
    assert ids[4].tolist() == [0, 1, 2, 3] and ids[5].tolist() == [0, 1, 2, 3] and (w[5] == 0.25).all()
    assert ids[6].tolist() == [38, 39, -1, -1] and w[6].tolist() == [0.5, 0.5, 0, 0]
    check_sort(p, ids, 40)


@pytest.mark.parametrize("n,e,k", [(0, 8, 2), (1, 1, 16), (64, 3, 16), (65, 3, 16), (1000, 1024, 16), (5000, 7, 1), (30000, 128, 8)])
def test_sort_of_given_ids(dev, n, e, k):
    g = torch.Generator(device=dev).manual_seed(n)
    ids = torch.randint(-2, e + 2, (n, k), dtype=torch.int32, device=dev, generator=g)  # some none, some twice
    if n > 70:
        ids[7:50] = 0                             # a stretch of one expert
    w = torch.rand(n, k, device=dev, generator=g) + 0.5
    p = sg.MoePlan(n + 1, k, e, device=dev)
    for _ in range(2):
        sg.moe_sort(ids, w, p)
        there = (ids >= 0) & (ids < e)
        assert torch.equal(p.ids, torch.where(there, ids, -1)) and torch.equal(p.weights, torch.where(there, w, 0))
        check_sort(p, ids, e)


def test_nothing_to_sort(dev):
    p = sg.moe_route(torch.zeros(0, 32, device=dev), sg.MoePlan(10, 4, 32, device=dev))
    assert p.ids.shape == (0, 4) and p.first.tolist() == [0] * 33
    w = sg.mx4_quantize(rand(dev, 32, 64, 64))
    assert sg.mx4_experts(torch.zeros(0, 64, device=dev), w, p).shape == (0, 64)
    assert sg.moe_combine(torch.zeros(0, 64, device=dev), p).shape == (0, 64)
    # tokens without any expert: no product, zeros back
    p = sg.moe_route(torch.full((5, 32), float("-inf"), device=dev), sg.MoePlan(10, 4, 32, device=dev))
    x = rand(dev, 5, 64)
    y = torch.full((20, 64), 7.0, device=dev)
    sg.mx4_experts(x, w, p, gather=True, out=y)
    assert (y == 7).all() and sg.moe_combine(y, p).count_nonzero() == 0 and (p.order == -1).all()
    with pytest.raises(sg.SgError):
        sg.moe_combine(y, p, out=y[:5])           # over its own input


def test_plans_are_used_again(dev):
    p = sg.MoePlan(3000, 4, 32, device=dev)
    for n in (3000, 5, 0, 64, 2999):
        ids = torch.randint(0, 32, (n, 4), dtype=torch.int32, device=dev)
        sg.moe_sort(ids, torch.ones(n, 4, device=dev), p)
        assert p.ids.shape == (n, 4) and p.order.shape == (4 * n,)
        check_sort(p, ids, 32)
    with pytest.raises(ValueError):
        sg.moe_route(torch.zeros(3001, 32, device=dev), p)
    with pytest.raises(ValueError):
        sg.moe_route(torch.zeros(30, 31, device=dev), p)
    with pytest.raises(ValueError):
        sg.moe_sort(torch.zeros(30, 3, dtype=torch.int32, device=dev), torch.zeros(30, 3, device=dev), p)
    with pytest.raises(TypeError):
        sg.moe_sort(torch.zeros(30, 4, dtype=torch.int64, device=dev), torch.zeros(30, 4, device=dev), p)


def experts_one_by_one(x, ws, first):
    """Results and bounds of the rows sorted by expert, [places, rows] of x's quantized rows."""
    out, bound = [], []
    for e in range(len(first) - 1):
        y, b = U.product(x[first[e]:first[e + 1]], *[w[e] for w in ws])
        out.append(y), bound.append(b)
    return torch.cat(out), torch.cat(bound)


@pytest.mark.parametrize("n,e,k,dim,ff", [(1, 8, 2, 256, 128), (1, 128, 8, 512, 96), (5, 4, 4, 96, 300), (16, 64, 6, 1024, 130), (40, 3, 2, 512, 200),
                                          (100, 128, 8, 256, 64), (333, 8, 2, 544, 257), (1500, 5, 3, 256, 128), (2000, 32, 1, 288, 96)])
def test_experts_and_back(dev, n, e, k, dim, ff):
    x, logits = rand(dev, n, dim, seed=n), rand(dev, n, e, seed=1) * 2
    logits[:, 0] = float("-inf")                  # an expert that no token reaches
    gate, up, down = rand(dev, e, ff, dim, seed=2) * dim ** -0.5, rand(dev, e, ff, dim, seed=3) * dim ** -0.5, rand(dev, e, dim, ff // 32 * 32, seed=4) * ff ** -0.5
    G, V, D = (sg.mx4_quantize(t) for t in (gate, up, down))
    gq, vq, dq = (U.quantized(t) for t in (gate, up, down))
    p = sg.moe_route(logits, sg.MoePlan(n, k, e, device=dev))
    used = int(p.first[-1])
    first, order, place = p.first.tolist(), p.order[:used].long(), p.place.long()
    for dtype in TYPES:
        t = x.to(dtype)
        out = torch.full((n * k, ff), 7.0, dtype=dtype, device=dev)
        h = sg.mx4_experts(t, G, p, up=V, out=out)
        want, bound = experts_one_by_one(U.quantized(t)[order // k], (gq, vq), first)
        assert U.close(h[:used], want, bound) and (h[used:] == 7).all()
        plain = sg.mx4_experts(t, G, p, gather=True)
        assert U.close(plain[:used], *experts_one_by_one(U.quantized(t)[order // k], (gq,), first))
        hs = h[:, :ff // 32 * 32]                 # (rows of another stride where ff is no multiple of 32)
        y = sg.mx4_experts(hs, D, p, dtype=torch.float32)
        assert U.close(y[:used], *experts_one_by_one(U.quantized(hs[:used].contiguous()), (dq,), first))
        o = sg.moe_combine(y, p, dtype=dtype)
        z = torch.where(place[..., None] < 0, 0.0, y[place.clamp(min=0)].double()) * p.weights[..., None].double()
        assert U.close(o, z.sum(1), z.abs().sum(1) * (k * 2.0 ** -24))
    sg.device_status()


def test_experts_given_twice_and_crowded(dev):
    # all tokens at one expert, one of them twice
    n, e = 700, 6
    ids = torch.full((n, 2), 3, dtype=torch.int32, device=dev)
    ids[:, 1] = -1
    ids[10, 1] = 3
    p = sg.moe_sort(ids, torch.ones(n, 2, device=dev), sg.MoePlan(n, 2, e, device=dev))
    x, w = rand(dev, n, 256, seed=1), rand(dev, e, 200, 256, seed=2) * 0.06
    y = sg.mx4_experts(x, sg.mx4_quantize(w), p, gather=True)
    want, bound = U.product(U.quantized(x), U.quantized(w[3]))
    o = sg.moe_combine(y, p)
    twice = torch.ones(n, 1, device=dev, dtype=torch.float64)
    twice[10] = 2
    assert U.close(o, want * twice, (bound + want.abs() * 2.0 ** -24) * twice)
    with pytest.raises(ValueError):
        sg.mx4_experts(x, sg.mx4_quantize(w[:5]), p, gather=True)
    with pytest.raises(ValueError):
        sg.mx4_experts(x, sg.mx4_quantize(w), p)  # rows sorted by expert are wanted


@pytest.mark.parametrize("dim", [1, 7, 8, 33, 512, 1000])
@pytest.mark.parametrize("k", [1, 3, 8, 11, 16])
def test_combine(dev, dim, k):
    n = 50
    ids = torch.randint(-1, 9, (n, k), dtype=torch.int32, device=dev, generator=torch.Generator(device=dev).manual_seed(k))
    ids[4] = -1
    p = sg.moe_sort(ids, rand(dev, n, k, seed=5), sg.MoePlan(n, k, 8, device=dev))
    base = rand(dev, n * k, dim + 3, seed=6)
    base[int(p.first[-1]):] = float("nan")        # places that no pair has
    place = p.place.long()
    for dtype in TYPES:
        for off in (0, 1):
            y = base.to(dtype)[:, off:off + dim]
            z = torch.where(place[..., None] < 0, 0.0, y[place.clamp(min=0)].double() * p.weights[..., None].double())
            for ot in TYPES:
                out = torch.full((n, dim + 2), 7.0, dtype=ot, device=dev)
                sg.moe_combine(y, p, out=out[:, 1:1 + dim])
                assert U.close(out[:, 1:1 + dim], z.sum(1), z.abs().sum(1) * (k * 2.0 ** -24))
                assert (out[:, 0] == 7).all() and (out[:, -1] == 7).all() and (out[4, 1:-1] == 0).all()


@pytest.mark.parametrize("n,dim", [(1, 8), (3, 1000), (701, 1192)])
@pytest.mark.parametrize("k", [1, 2, 4, 5, 8, 16])
def test_combine_whole_rows(dev, n, dim, k):
    # rows of 16-byte words, several of them a thread where a token has few
    ids = torch.randint(-1, 20, (n, k), dtype=torch.int32, device=dev, generator=torch.Generator(device=dev).manual_seed(k))
    p = sg.moe_sort(ids, rand(dev, n, k, seed=5), sg.MoePlan(n, k, 20, device=dev))
    base = rand(dev, n * k, dim, seed=6)
    base[int(p.first[-1]):] = float("nan")
    place = p.place.long()
    for dtype in TYPES:
        y = base.to(dtype)
        z = torch.where(place[..., None] < 0, 0.0, y[place.clamp(min=0)].double() * p.weights[..., None].double())
        for ot in TYPES:
            out = torch.full((n + 1, dim + 8), 7.0, dtype=ot, device=dev)
            sg.moe_combine(y, p, out=out[:-1, :dim])
            assert U.close(out[:-1, :dim], z.sum(1), z.abs().sum(1) * (k * 2.0 ** -24))
            assert (out[-1] == 7).all() and (out[:, dim:] == 7).all()


def test_captured_layer(dev):
    # route, experts and back in one graph, replayed with other tokens
    n, e, k, dim, ff = 24, 16, 4, 256, 128
    x, router = rand(dev, n, dim), rand(dev, e, dim, seed=1) * 0.1
    G, V, D = (sg.mx4_quantize(rand(dev, e, a, b, seed=s) * 0.06) for a, b, s in ((ff, dim, 2), (ff, dim, 3), (dim, ff, 4)))
    plans = [sg.MoePlan(n, k, e, device=dev) for _ in range(2)]

    def layer(p, s):
        sg.moe_route(x @ router.T, p)
        return sg.moe_combine(sg.mx4_experts(sg.mx4_experts(x, G, p, up=V, scratch=s[0]), D, p, scratch=s[1]), p)
    sg.moe_route(x @ router.T, plans[0])
    bufs = [tuple(sg.mx4_scratch(m, plans[0]) for m in (G, D)) for _ in range(2)]
    layer(plans[0], bufs[0])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = layer(plans[0], bufs[0])
    for seed in (5, 6):
        x.copy_(rand(dev, n, dim, seed=seed))
        g.replay()
        assert torch.equal(got, layer(plans[1], bufs[1]))
    sg.device_status()
