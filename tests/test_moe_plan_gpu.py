"""Plans of tokens sorted by expert on the GPU: what they hold after refused calls, and their use
for steps of other sizes."""
import pytest
import torch

import spindle_b200 as sg
from spindle_b200.mx4 import _scratch_bytes

pytestmark = pytest.mark.gpu


def rand(dev, *shape, seed=0):
    return torch.randn(*shape, device=dev, generator=torch.Generator(device=dev).manual_seed(seed))


@pytest.mark.parametrize("n,other", [(300, 5), (5, 300), (70, 69)])
def test_refused_calls_leave_the_plan(dev, n, other):
    e, k = 12, 3
    x, w = rand(dev, n, 64, seed=1), sg.mx4_quantize(rand(dev, e, 40, 64, seed=2))
    p = sg.moe_route(rand(dev, n, e, seed=3), sg.MoePlan(400, k, e, device=dev))
    held = [t.clone() for t in (p.ids, p.weights, p.first, p.order, p.place)]
    want = sg.moe_combine(sg.mx4_experts(x, w, p, gather=True), p)
    ids, logits = torch.zeros(other, k, dtype=torch.int32, device=dev), rand(dev, other + 1, e + 1, seed=4)
    for call in (lambda: sg.moe_sort(ids.long(), ids.float(), p), lambda: sg.moe_sort(ids.T.contiguous().T, ids.float(), p),
                 lambda: sg.moe_sort(ids, ids.double(), p), lambda: sg.moe_route(logits[:other], p), lambda: sg.moe_route(logits[:other, :e].double(), p),
                 lambda: sg.moe_route(logits[:1, :e].expand(other, e), p),                       # rows one over the other
                 lambda: sg.moe_route(torch.zeros(401, e, device=dev), p), lambda: sg.moe_route(logits[:other, :e], p, prune="none")):
        with pytest.raises((TypeError, ValueError, sg.SgError)):
            call()
        assert p.n_tok == n and p.ids.shape == (n, k) and p.order.shape == (n * k,)
        for t, was in zip((p.ids, p.weights, p.first, p.order, p.place), held):
            assert torch.equal(t, was)
        assert torch.equal(sg.moe_combine(sg.mx4_experts(x, w, p, gather=True), p), want)
    sg.device_status()


@pytest.mark.parametrize("e,k,most", [(8, 2, 700), (128, 8, 600)])
def test_one_scratch_for_all_steps(dev, e, k, most):
    # made beside the plan, before any step; kept as the steps grow and shrink
    w = sg.mx4_quantize(rand(dev, e, 200, 320, seed=2))
    p = sg.MoePlan(most, k, e, device=dev)
    scratch, rows = sg.mx4_scratch(w, p), sg.mx4_scratch(sg.mx4_quantize(rand(dev, 200, 320)), most)
    for n in (0, 5, most, 33, 300, 1):
        x = rand(dev, n, 320, seed=n)
        sg.moe_route(rand(dev, n, e, seed=n + 1), p)
        assert torch.equal(sg.mx4_experts(x, w, p, gather=True, scratch=scratch), sg.mx4_experts(x, w, p, gather=True))
        assert sg.mx4_scratch(w, p).numel() == scratch.numel()
        W = sg.mx4_quantize(rand(dev, 200, 320, seed=3))
        assert torch.equal(sg.mx4_matmul(x, W, scratch=rows), sg.mx4_matmul(x, W))
    sg.device_status()


@pytest.mark.parametrize("n,first", [(6000, 1), (6000, 2999), (90, 37)])
def test_sort_of_the_plans_own_arrays(dev, n, first):
    ids = torch.randint(-1, 16, (n, 4), dtype=torch.int32, device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    w = rand(dev, n, 4, seed=2)
    a, b = (sg.moe_sort(ids, w, sg.MoePlan(n, 4, 16, device=dev)) for _ in range(2))
    sg.moe_sort(a.ids[first:], a.weights[first:], a)
    sg.moe_sort(ids[first:].clone(), b.weights[first:].clone(), b)
    for x, y in ((a.ids, b.ids), (a.weights, b.weights), (a.first, b.first), (a.order, b.order), (a.place, b.place)):
        assert torch.equal(x, y)
    assert torch.equal(a.ids, ids[first:])


def test_read_back_between_rows(dev):
    # an expert's rows behind the other's, and all experts' between two rows
    x = rand(dev, 3, 70, 96, seed=1)
    m = sg.mx4_quantize(x)
    want = sg.mx4_dequantize(m)
    for out in (torch.full((3, 75, 100), 7.0, device=dev)[:, :70, :96], torch.full((70, 3, 99), 7.0, device=dev).transpose(0, 1)[:, :, :96],
                torch.full((70, 3, 96), 7.0, device=dev).transpose(0, 1)):
        assert torch.equal(sg.mx4_dequantize(m, out=out), want)
    with pytest.raises(sg.SgError):
        sg.mx4_dequantize(m, out=torch.zeros(1, 70, 96, device=dev).expand(3, 70, 96))


@pytest.mark.parametrize("e,k,many,few,ff", [(16, 2, 3000, 40, 200), (16, 2, 3000, 2500, 200), (64, 4, 2000, 300, 1300), (4, 1, 900, 1, 64)])
def test_a_plan_filled_by_a_replayed_graph(dev, e, k, many, few, ff):
    # a graph sorts other numbers of tokens into the plan than the last call did that the host made: what the products give is
    # not defined then, but they write into their rows and scratch only
    dim = 320
    w, v, d = (sg.mx4_quantize(rand(dev, e, a, b, seed=s) * 0.05) for a, b, s in ((ff, dim, 1), (ff, dim, 2), (dim, ff // 32 * 32, 3)))
    p = sg.MoePlan(many, k, e, device=dev)
    skew = rand(dev, e, seed=4) * 2
    graphs = {}
    for n in (many, few):
        logits = rand(dev, n, e, seed=n) + skew
        sg.moe_route(logits, p)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            sg.moe_route(logits, p)
        graphs[n] = g, logits
    for n, other in ((few, many), (many, few)):
        sg.moe_route(graphs[n][1], p)
        graphs[other][0].replay()                 # p.n_tok is n, the arrays hold other tokens
        rows, x = n * k, rand(dev, n, dim, seed=5)
        h = rand(dev, n * k, ff // 32 * 32, seed=6)
        for m, call in ((w, lambda o, s: sg.mx4_experts(x, w, p, up=v, out=o, scratch=s)),           # noqa: B023
                        (w, lambda o, s: sg.mx4_experts(x, w, p, gather=True, out=o, scratch=s)),    # noqa: B023
                        (d, lambda o, s: sg.mx4_experts(h, d, p, out=o, scratch=s))):                # noqa: B023
            size = _scratch_bytes(m, 0, p._c)
            out, scratch = torch.full((rows + 4000, m.rows), 7.0, device=dev), torch.full((size + (1 << 22),), 0x5A, dtype=torch.uint8, device=dev)
            call(out[:rows], scratch[:size])
            assert (out[rows:] == 7).all() and (scratch[size:] == 0x5A).all()
        y = torch.full((n + 4000, dim), 7.0, device=dev)
        sg.moe_combine(rand(dev, rows, dim, seed=7), p, out=y[:n])
        assert (y[n:] == 7).all()
        # filled for its own tokens again, all is as it was
        graphs[n][0].replay()
        got = sg.mx4_experts(x, w, p, gather=True)
        q = sg.moe_route(graphs[n][1], sg.MoePlan(n, k, e, device=dev))
        assert torch.equal(sg.moe_combine(got, p), sg.moe_combine(sg.mx4_experts(x, w, q, gather=True), q))
    sg.device_status()
