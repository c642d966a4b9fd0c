"""The paged 4-bit KV cache on the GPU at the edges of what its entry points take."""
import random

import pytest
import torch

import kv4_util as U
import spindle_b200 as sg
from test_kv4_gpu import ROUND, TYPES, U24, case, check, ints

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


def finite_quantized(x):
    """kv4_util.quantized with the step that keeps a group's largest value finite in f16: one f16 step
    less where m + 15 s, in f32, is 65520 or more."""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=U.F16_MAX, neginf=-U.F16_MAX).clamp(-U.F16_MAX, U.F16_MAX)
    g = x.unflatten(-1, (x.shape[-1] // 32, 32))
    m = g.amin(-1, keepdim=True).half().float()
    s = ((g.amax(-1, keepdim=True) - m).clamp(min=0) * torch.tensor(1.0 / 15.0)).half()
    less = (s.view(torch.int16) - 1).view(torch.float16)
    s = torch.where(m.double() + 15 * s.double() >= 65520.0 - 2.0 ** -9, less, s).float()
    r = torch.where(s > 0, torch.tensor(1.0) / s, torch.zeros(()))
    c = torch.round(((g - m) * r).clamp(0, 15))
    return (m.double() + s.double() * c.double()).flatten(-2)


def full_range(n, heads, d, dtype, seed):
    """Rows whose groups reach f16's ends: from 0 or a little above to infinity, from one infinity to the other, and ordinary ones."""
    g = torch.Generator().manual_seed(seed)
    inf = float("inf")
    x = torch.randn(n, heads, d, generator=g)
    x[0, 0, :32] = x[0, 0, :32].abs()
    x[0, 0, 3] = inf                     # 0.. to the largest
    x[1, 0, :32], x[1, 0, 9] = 0.0, 65504.0
    x[2, 0, :32] = 14.0
    x[2, 0, 31] = inf
    x[3, 0, 32:64] = x[3, 0, 32:64] * 100
    x[3, 0, 40], x[3, 0, 41] = inf, -inf
    x[4, 0, 5], x[4, 0, 6] = -inf, 60000.0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,heads,page", [(64, 1, 16), (128, 2, 32), (256, 1, 64)])
def test_append_holds_what_is_finite_in_f16(dev, dtype, d, heads, page):
    n = 40
    x = full_range(n, heads, d, dtype, d)
    cache = sg.Kv4Cache(64 // page + 2, heads, d, page, device=dev)
    slots = torch.arange(n, dtype=torch.int32, device=dev)
    sg.kv4_append(cache, x.to(dev), x.to(dev), slots)
    want = finite_quantized(x.float())
    for out_type in TYPES:
        for t in sg.kv4_read(cache, slots, dtype=out_type):
            assert torch.isfinite(t).all()
            assert torch.equal(t.cpu(), want.float().to(out_type))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group,new", [(2, 3), (8, 300), (8, 1500)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_over_the_whole_range_of_f16(dev, dtype, group, new, d):
    # a few positions with such rows among ordinary ones: finite results, right against 64 bits, and the rows that do not
    # see those positions have the bits that they have without them
    heads, page, length = 2, 16, 1600
    cache, ref = (sg.Kv4Cache(length // page, heads, d, page, device=dev) for _ in range(2))
    slots = torch.arange(length, dtype=torch.int32, device=dev)
    g = torch.Generator(device=dev).manual_seed(5)
    k = torch.randn(length, heads, d, device=dev, generator=g)
    v = torch.randn(length, heads, d, device=dev, generator=g)
    sg.kv4_append(ref, k, v, slots)
    at = length - 10
    k[at:at + 5, :1] = full_range(5, 1, d, torch.float32, 1).to(dev)
    v[at:at + 5, :1] = full_range(5, 1, d, torch.float32, 2).to(dev)
    sg.kv4_append(cache, k, v, slots)
    tables = torch.arange(length // page, dtype=torch.int32, device=dev)[None]
    q = torch.randn(new, heads * group, d, device=dev, generator=g).to(dtype)
    cu, seq = ints([0, new], dev), ints([length], dev)
    out = sg.kv4_attention(cache, q, cu, seq, tables)
    check(dev, cache, tables, tables.cpu(), cu, seq, q, d ** -0.5, 0, out, None)
    want = sg.kv4_attention(ref, q, cu, seq, tables)
    before = torch.arange(length - new, length, device=dev) < at
    assert torch.equal(out[:, group:], want[:, group:])
    if before.any() and dtype != torch.float32:
        assert torch.equal(out[before], want[before])
    elif before.any():
        # f32 holds the sums of a group at a power of two for its largest scale, 2^14 times the ordinary ones here: a
        # position's weight times value is off by up to 8 * 2^-25 * 2^6 of the largest weight, 1600 of them over a sum
        # of weights that is at least 25 for these scores
        assert (out[before] - want[before]).abs().max() <= 1600 * 8 * 2.0 ** -19 / 25


def test_plan_captured_with_its_own_ring(dev):
    # a captured plan on the plan's own ring goes on from replay to replay, over page ends, and calls outside the graph go on from there
    n, page, n_blocks, width = 3, 16, 40, 12
    plan = sg.Kv4Plan(n, 8, page, n_blocks, device=dev)
    tables = torch.full((n, width), -1, dtype=torch.int32, device=dev)
    ctx, new = ints([0] * n, dev), ints([1, 2, 0], dev)
    side = torch.cuda.Stream()
    want_t, ring, head, tail = [[-1] * width for _ in range(n)], list(range(n_blocks)), 0, n_blocks
    lens, graph = [0] * n, None
    for t in range(70):
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            if t == 3:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    sg.kv4_plan(plan, ctx, new, tables)
            if graph is None or t % 10 == 9:
                sg.kv4_plan(plan, ctx, new, tables)
            else:
                graph.replay()
        torch.cuda.synchronize()
        want = U.plan(lens, [1, 2, 0], want_t, ring, head, tail, page, n_blocks, 8)
        assert [x.tolist() for x in (plan.cu, plan.seq, plan.pos, plan.slots, plan.info)] == [list(x) for x in want], t
        assert tables.tolist() == want_t and plan.ring.tolist() == ring, t
        head, tail = want[4][:2]
        lens = want[1]
        ctx.copy_(plan.seq)
    del graph


def test_plan_own_and_given_rings_apart(dev):
    # calls with a ring and cursor of the caller leave the plan's own ones as they are, and infos feed the next call
    plan = sg.Kv4Plan(1, 40, 16, 6, device=dev)
    tables = [torch.full((1, 8), -1, dtype=torch.int32, device=dev) for _ in range(2)]
    ring, cursor = torch.arange(6, dtype=torch.int32, device=dev).flip(0).contiguous(), ints([2, 8], dev)
    want_t, want_r, at = [[[-1] * 8], [[-1] * 8]], [list(range(6)), ring.tolist()], [(0, 6), (2, 8)]
    for step, (own, ctx) in enumerate([(True, 0), (False, 0), (False, 20), (True, 20), (False, 40), (True, 40)]):
        k = 0 if own else 1
        got = sg.kv4_plan(plan, ints([ctx], dev), ints([20], dev), tables[k], *(() if own else (ring, cursor)))
        want = U.plan([ctx], [20], want_t[k], want_r[k], *at[k], 16, 6, 40)
        assert got.info.tolist() == list(want[4]) and tables[k].tolist() == want_t[k], step
        at[k] = want[4][:2]
        if not own:
            cursor = got.info                              # the tensor itself, or a copy of it
            if step == 1:
                cursor = cursor[:2].clone()


@pytest.mark.parametrize("n_req,most,page,n_blocks", [(3, 9, 16, 40), (5, 5000, 1024, 64), (1500, 40, 16, 20000), (64, 300, 64, 2000)])
def test_plan_lengths_in_place(dev, n_req, most, page, n_blocks):
    # plan.seq as the next call's lengths: steps of one CTA and of many
    rng = random.Random(n_req)
    width = (4 * most + page - 1) // page + 3
    cap = n_req * most + 5
    plan = sg.Kv4Plan(n_req, cap, page, n_blocks, device=dev)
    plan.seq.zero_()
    tables = torch.full((n_req, width), -1, dtype=torch.int32, device=dev)
    want_t, ring, at, ctx = [[-1] * width for _ in range(n_req)], list(range(n_blocks)), (0, n_blocks), [0] * n_req
    for step in range(4):
        new = [-1 if step and rng.random() < 0.2 else rng.choice([0, 1, most]) for _ in range(n_req)]
        sg.kv4_plan(plan, plan.seq, ints(new, dev), tables)
        want = U.plan(ctx, new, want_t, ring, *at, page, n_blocks, cap)
        for a, b in zip((plan.cu, plan.seq, plan.pos, plan.slots, plan.info), want):
            assert a.tolist() == list(b)
        assert tables.tolist() == want_t and plan.ring.tolist() == ring
        at, ctx = want[4][:2], want[1]


def test_plan_refuses_what_it_would_overwrite(dev):
    plan = sg.Kv4Plan(2, 4, 16, 4, device=dev)
    z, t = ints([0, 0], dev), torch.full((2, 2), -1, dtype=torch.int32, device=dev)
    for ctx, new in ((plan.cu[:2], z), (plan.cu[1:], z), (z, plan.seq), (plan.pos[2:], z), (z, plan.slots[:2]), (plan.ring[1:3], z),
                     (t[0], z), (z, t[1])):
        with pytest.raises(sg.SgError):
            sg.kv4_plan(plan, ctx, new, t)
    for cursor in (plan.cu, plan.seq, plan.pos, plan.ring):
        with pytest.raises(sg.SgError):
            sg.kv4_plan(plan, z, z, t, plan.ring, cursor)
    sg.kv4_plan(plan, z, z, t)
    # side by side in one buffer is fine
    buf = torch.zeros(16, dtype=torch.int32, device=dev)
    buf[4:6] = ints([0, 4], dev)
    plan.ring = torch.arange(4, dtype=torch.int32, device=dev)
    sg.kv4_plan(plan, buf[0:2], buf[2:4], buf[12:16].view(2, 2), plan.ring, buf[4:6])
    assert plan.seq.tolist() == [0, 0]


def flat_tail(dev, n, k, heads, d, sink_v):
    """A key 2^k ahead (for q = e_0) of n - 1 equal ones: cache, tables of one row, and the two keys and values in 64 bits
    as the cache holds them.  All positions after the first page lie in one block."""
    page = 64
    cache = sg.Kv4Cache(2, heads, d, page, device=dev)
    g = torch.Generator(device=dev).manual_seed(2)
    key = torch.randn(2, heads, d, device=dev, generator=g)
    v = torch.randn(2, heads, d, device=dev, generator=g).abs() + 0.5
    key[0] = key[1]
    key[0, :, 0] += 8.0
    v[0] = v[0] if sink_v is None else sink_v
    rows = [torch.cat([t[:1], t[1:].expand(2 * page - 1, heads, d)]) for t in (key, v)]
    sg.kv4_append(cache, *rows, torch.arange(2 * page, dtype=torch.int32, device=dev))
    tables = torch.ones(1, (n + page - 1) // page, dtype=torch.int32, device=dev)
    tables[:, 0] = 0
    kk, vv = (t.double() for t in sg.kv4_read(cache, ints([0, page], dev), dtype=torch.float32))
    scale = torch.tensor(k * 0.6931471805599453 / (kk[0, 0, 0] - kk[1, 0, 0]).item(), dtype=torch.float32).item()
    w = torch.exp(scale * (kk[1, :, 0] - kk[0, :, 0]))[:, None] * (n - 1)   # of all the equal ones, by heads
    return cache, tables, scale, (vv[0] + w * vv[1]) / (1 + w), scale * kk[0, :, 0] + torch.log1p(w[:, 0]), vv


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,k", [(1024, 10), (4096, 12), (16384, 14)])
def test_attention_f32_first_token_and_a_flat_tail(dev, n, k, d):
    # a first key that weighs as much as all the others together, and a request per warp, so that one running sum takes
    # all of it: n / 16 rounded additions of values, n / 32 of weights, half a unit in the last place each, and some
    # for the scores, weights and products
    heads, n_req = 2, 1024
    cache, tables, scale, want, wl, vv = flat_tail(dev, n, k, heads, d, None)
    q = torch.zeros(n_req, heads, d, device=dev)
    q[:, :, 0] = 1.0
    cu, seq = torch.arange(n_req + 1, dtype=torch.int32, device=dev), torch.full((n_req,), n, dtype=torch.int32, device=dev)
    lse = torch.empty(n_req, heads, device=dev)
    out = sg.kv4_attention(cache, q, cu, seq, tables.repeat(n_req, 1), scale=scale, max_new=1, lse=lse)
    assert ((out.double() - want).abs() / vv.amax()).max() <= (n / 16 + n / 32 + 64) * U24
    assert (lse.double() - wl).abs().max() <= (n / 32 + 64) * U24


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 900])
@pytest.mark.parametrize("d,k", [(64, 12), (64, 16), (64, 20), (128, 16), (256, 20)])
def test_attention_weights_far_below_the_largest(dev, dtype, d, k, new):
    # the first key has nearly all the weight and a value of zeros: the result is the others' alone, each 2^-k of the
    # largest.  A weight keeps 25 + 12 - k bits in f32, where its product with a scale is rounded once more, and at
    # least 2^-12 in the 16-bit types (either kernel), besides V's rounding and the result's; scores below 32 in base
    # 2 are known to three times 2^-20 times ln 2; n / 16 additions of values and n / 32 of weights in a warp at most.
    # f32 sums (c - 8) s and m + 8 s apart: 8 / 15 of a group's span and a value, below 3 times the largest value
    heads, group, n = 4, 8, 900 + new
    cache, tables, scale, want, _, vv = flat_tail(dev, n, k, heads, d, 0.0)
    q = torch.zeros(new, heads * group, d, device=dev, dtype=dtype)
    q[..., 0] = 1.0
    out = sg.kv4_attention(cache, q, ints([0, new], dev), ints([n], dev), tables, scale=scale)[-1]
    share = (want / vv[1]).repeat_interleave(group, 0)                # of the weight that the others have
    want = want.repeat_interleave(group, 0)
    tol = 2.0 ** (k - 36) + 3 * 2.0 ** -20 + (n / 16 + n / 32 + 64) * U24
    if dtype != torch.float32:
        tol += 2.0 ** -12 + 2.0 ** -11 + ROUND[dtype]
    assert ((out.double() - want).abs() <= tol * 3 * vv.amax() * share).all()


def test_attention_f32_is_f32(dev):
    # the root mean square of the errors in f32, where roundings meet in quadrature: scores that are off by
    # sqrt(d) 2^-24 of sum |q k| (about 4), weights and their products by 2^-22 of the largest, sums by less
    for heads, group, d, lens, news in [(2, 4, 64, [3000, 17], [1, 9]), (4, 8, 128, [5000, 900, 1], [1, 1, 1]), (8, 2, 128, [2050] * 4, [9] * 4),
                                        (2, 4, 256, [700, 300], [200, 130]), (1, 7, 128, [70000], [2])]:
        cache, tables, full, cu, seq, g = case(dev, lens, news, heads, d, 64, d)
        q = torch.randn(sum(news), heads * group, d, device=dev, generator=g)
        out = sg.kv4_attention(cache, q, cu, seq, tables, max_new=max(news)).double()
        off, norm = 0.0, 0.0
        for i, length in enumerate(lens):
            a, b = cu[i].item(), cu[i + 1].item()
            pos = torch.arange(length)
            slots = (full[i][pos // 64] * 64 + pos % 64).int().to(dev)
            k, v = (t.double() for t in sg.kv4_read(cache, slots, dtype=torch.float32))
            want, _, _ = U.attention(q[a:b].double(), k, v, torch.arange(length - (b - a), length, device=dev),
                                     torch.ones(length, dtype=torch.bool, device=dev), d ** -0.5, 0)
            off, norm = off + (out[a:b] - want).pow(2).sum().item(), norm + want.pow(2).sum().item()
        assert (off / norm) ** 0.5 <= 4 * d ** 0.5 * U24 + 2.0 ** -21, (d, lens, (off / norm) ** 0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_tok,heads,group", [(9, 2, 4), (1500, 4, 8)])
def test_attention_tokens_before_the_first_request(dev, dtype, n_tok, heads, group):
    # a part of the requests: the tokens before and after theirs belong to none
    lens = [300, 77, 40]
    a, b, c = n_tok // 3, n_tok // 3 * 2, n_tok - 1
    cache, tables, full, _, seq, g = case(dev, [max(l, n_tok) for l in lens[:2]], [1, 1], heads, 64, 16, 4)
    cu = ints([a, b, c], dev)
    q = torch.randn(n_tok, heads * group, 64, device=dev, generator=g).to(dtype)
    out = torch.full_like(q, 7.0)
    lse = torch.full((n_tok, heads * group), 7.0, device=dev)
    sg.kv4_attention(cache, q, cu, seq, tables, out=out, lse=lse)
    check(dev, cache, tables, full, cu, seq, q, 64 ** -0.5, 0, out, lse)
    for none in (slice(0, a), slice(c, n_tok)):
        assert (out[none] == 0).all() and torch.isneginf(lse[none]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_more_new_tokens_than_max_new(dev, dtype, d):
    # a bound that is too small: every row is written, right up to the bound, and right or NaN past it
    lens, news, heads, group = [700, 400], [600, 2], 4, 8
    cache, tables, full, cu, seq, g = case(dev, lens, news, heads, d, 16, 8)
    q = torch.randn(sum(news), heads * group, d, device=dev, generator=g).to(dtype)
    right, rl = torch.empty_like(q), torch.empty(sum(news), heads * group, device=dev)
    sg.kv4_attention(cache, q, cu, seq, tables, out=right, lse=rl)
    for bound in (1, 100, 599):
        out, lse = torch.full_like(q, 7.0), torch.full_like(rl, 7.0)
        sg.kv4_attention(cache, q, cu, seq, tables, out=out, lse=lse, max_new=bound)
        nan = torch.isnan(out)
        assert torch.equal(nan[..., 0], torch.isnan(lse)) and torch.equal(nan, nan[..., :1].expand_as(nan))
        assert not nan[:bound].any() and not nan[600:].any() if bound > 1 else not nan[:1].any()
        assert torch.equal(out[~nan], right[~nan]) and torch.equal(lse[~nan[..., 0]], rl[~nan[..., 0]])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 3, 700])
def test_attention_tiny_scales(dev, dtype, new):
    # scales so small that they and the smallest query's power of two leave f32's range: equal weights
    heads, group, d, lens = 4, 8, 64, [new + 5, new, 800]
    cache, tables, full, cu, seq, g = case(dev, lens, [new] * 3, heads, d, 16, new)
    q = torch.randn(3 * new, heads * group, d, device=dev, generator=g)
    q[0] = 0
    q[1, ::2] *= 1e-30
    q = q.to(dtype)
    for scale in (1e-20, 1e-38, -1e-44):
        lse = torch.empty(3 * new, heads * group, device=dev)
        out = sg.kv4_attention(cache, q, cu, seq, tables, scale=scale, lse=lse, max_new=new)
        check(dev, cache, tables, full, cu, seq, q, scale, 0, out, lse)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_scale_of_zero(dev, dtype):
    # not the default: every seen position weighs the same
    cache, tables, full, cu, seq, g = case(dev, [100, 1], [1, 1], 2, 64, 16, 3)
    q = torch.randn(2, 8, 64, device=dev, generator=g).to(dtype)
    for zero in (0, 0.0, -0.0, 1e-60):
        check(dev, cache, tables, full, cu, seq, q, 0.0, 0, sg.kv4_attention(cache, q, cu, seq, tables, scale=zero), None)


@pytest.mark.parametrize("dtype,new", [(torch.float32, 1), (torch.float16, 1), (torch.float32, 9), (torch.bfloat16, 9), (torch.float16, 900),
                                       (torch.bfloat16, 900)])
@pytest.mark.parametrize("d,window", [(64, 100), (128, 1000), (256, 37)])
def test_attention_at_the_end_of_31_bits(dev, dtype, new, d, window):
    # the longest table there is, its last two blocks held: offsets of table entries, positions and steps near 2^31
    heads, group, page = 4, 8, 1024
    n = (1 << 31) - 1024
    cache = sg.Kv4Cache(2, heads, d, page, device=dev)
    g = torch.Generator(device=dev).manual_seed(window)
    k, v = (torch.randn(2 * page, heads, d, device=dev, generator=g) for _ in range(2))
    slots = torch.arange(2 * page, dtype=torch.int32, device=dev)
    sg.kv4_append(cache, k, v, slots)
    tables = torch.full((1, n // page), -1, dtype=torch.int32, device=dev)
    tables[0, -2:] = ints([0, 1], dev)
    q = torch.randn(new, heads * group, d, device=dev, generator=g).to(dtype)
    lse = torch.empty(new, heads * group, device=dev)
    out = sg.kv4_attention(cache, q, ints([0, new], dev), ints([n], dev), tables, window=window, lse=lse)
    check(dev, cache, ints([[0, 1]], dev), torch.tensor([[0, 1]]), ints([0, new], dev), ints([2 * page], dev), q, d ** -0.5, window, out, lse)
    sg.device_status()


@pytest.mark.parametrize("d,length,new", [(64, 2000, 900), (128, 3000, 700), (128, 8000, 300), (256, 1500, 700)])
def test_attention_f16_many_rows_keeps_its_bits(dev, d, length, new):
    # the root mean square error of a 16-bit result: a rounding to 11 bits is 2.1e-4 of a value (2^-10 / sqrt(12), over
    # mantissas from 1 to 2), and besides the result's there is the weights', in quadrature, where a few of them count
    # (the scale) and V has mean 0.  V's rounding would be a third: 3.6e-4
    heads, group, page = 4, 8, 32
    cache = sg.Kv4Cache((length + page - 1) // page, heads, d, page, device=dev)
    g = torch.Generator(device=dev).manual_seed(d)
    slots = torch.arange(length, dtype=torch.int32, device=dev)
    sg.kv4_append(cache, *(torch.randn(length, heads, d, device=dev, generator=g) for _ in range(2)), slots)
    tables = torch.arange(cache.n_blocks, dtype=torch.int32, device=dev)[None]
    q = torch.randn(new, heads * group, d, device=dev, generator=g).half()
    scale = 3 * d ** -0.5
    out = sg.kv4_attention(cache, q, ints([0, new], dev), ints([length], dev), tables, scale=scale).double()
    k, v = (t.double() for t in sg.kv4_read(cache, slots, dtype=torch.float32))
    want, _, _ = U.attention(q.double(), k, v, torch.arange(length - new, length, device=dev), torch.ones(length, dtype=torch.bool, device=dev),
                             scale, 0)
    off = ((out - want).norm() / want.norm()).item()
    assert off <= 2 ** 0.5 * 2.1e-4, off


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 7, 900])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("big", [1.0, 30.0, 1000.0, 3e4])
def test_attention_huge_scores(dev, dtype, new, d, big):
    # keys of infinities (held as f16's largest numbers) and large queries: scores of 1e5 to 1e10, whose last f32 bit is
    # worth more than a power of two of a weight.  The results are means of values all the same
    heads, group, length = 4, 8, 1000
    cache = sg.Kv4Cache(63, heads, d, 16, device=dev)
    g = torch.Generator(device=dev).manual_seed(d + new)
    k = torch.randn(length, heads, d, device=dev, generator=g)
    k[::3] *= 2e4
    k[5::50] = float("inf")
    k[6::70] = -float("inf")
    k[7::40, :, ::2] = float("inf")
    v = torch.randn(length, heads, d, device=dev, generator=g)
    sg.kv4_append(cache, k, v, torch.arange(length, dtype=torch.int32, device=dev))
    tables = torch.arange(63, dtype=torch.int32, device=dev)[None]
    q = (torch.randn(new, heads * group, d, device=dev, generator=g) * big).clamp(-65504, 65504).to(dtype)
    lse = torch.empty(new, heads * group, device=dev)
    out = sg.kv4_attention(cache, q, ints([0, new], dev), ints([length], dev), tables, lse=lse)
    check(dev, cache, tables, tables.cpu(), ints([0, new], dev), ints([length], dev), q, d ** -0.5, 0, out, lse)
    top = sg.kv4_read(cache, torch.arange(length, dtype=torch.int32, device=dev), dtype=torch.float32)[1].abs().amax()
    assert (out.abs() <= top * 1.05).all()
