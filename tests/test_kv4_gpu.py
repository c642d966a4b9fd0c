"""The paged 4-bit KV cache on the GPU (kv4_plan, kv4_append, kv4_read,
kv4_attention) against plain forms in 64 bits."""
import random

import pytest
import torch

import kv4_util as U
import spindle_b200 as sg

pytestmark = pytest.mark.gpu

U16, U8, U24 = 2.0 ** -11, 2.0 ** -8, 2.0 ** -24  # half a unit in the last place of f16, bf16 and f32, relative
ROUND = {torch.float32: U24, torch.float16: U16, torch.bfloat16: U8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# ---- plan ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("n_req,page,most,n_blocks", [(1, 16, 1, 8), (3, 16, 40, 64), (7, 64, 300, 40), (64, 16, 1, 4096),
                                                      (1500, 32, 50, 6000), (5, 1024, 5000, 64), (40, 16, 200, 100)])
def test_plan_steps(dev, n_req, page, most, n_blocks):
    # several steps in a row with the plan's own ring: requests come, grow, end and
    # come again; in the small caches blocks run out
    rng = random.Random(n_req * 7 + page)
    width = (4 * most + page - 1) // page + 3
    tables = [[-1] * width for _ in range(n_req)]
    ring, head, tail = list(range(n_blocks)), 0, n_blocks
    ctx = [0] * n_req
    cap = n_req * most + 5
    p = sg.Kv4Plan(n_req, cap, page, n_blocks, device=dev)
    t = ints(tables, dev)
    for step in range(4):
        new = [rng.choice([0, 1, rng.randint(0, most), most]) for _ in range(n_req)]
        if step:
            new = [-1 if rng.random() < 0.2 else a for a in new]
        got = sg.kv4_plan(p, ints(ctx, dev), ints(new, dev), t)
        want = U.plan(ctx, new, tables, ring, head, tail, page, n_blocks, cap)
        for a, b in zip((got.cu, got.seq, got.pos, got.slots, got.info), want):
            assert a.tolist() == list(b)
        assert t.tolist() == tables and p.ring.tolist() == ring
        head, tail = want[4][:2]
        ctx = want[1]


def test_plan_same_cursor_twice_and_table_strides(dev):
    n, page, n_blocks = 9, 16, 64
    wide = torch.full((n, 12), -7, dtype=torch.int32, device=dev)
    tables = wide[:, 2:9]
    ring = torch.randperm(n_blocks, device=dev).int()
    cursor = ints([60, 60 + 50, 99], dev)
    ctx, new = ints([0] * n, dev), ints([1, 0, 33, 16, 17, -1, 5, 100, 2], dev)
    p = sg.Kv4Plan(n, 200, page, n_blocks, device=dev)
    seen = []
    for _ in range(2):
        q = sg.kv4_plan(p, ctx, new, tables, ring, cursor)
        seen.append([x.tolist() for x in (q.cu, q.seq, q.pos, q.slots, q.info, wide, ring)])
    assert seen[0] == seen[1] and cursor.tolist() == [60, 110, 99]
    assert (wide[:, :2] == -7).all() and (wide[:, 9:] == -7).all()
    want_t = [[-7] * 7 for _ in range(n)]
    want = U.plan([0] * n, new.tolist(), want_t, ring.tolist(), 60, 110, page, n_blocks, 200)
    assert seen[0][:5] == [list(x) for x in want] and tables.tolist() == want_t


def test_plan_no_requests_and_no_tokens(dev):
    p = sg.Kv4Plan(0, 3, 16, 8, device=dev)
    e = torch.empty(0, dtype=torch.int32, device=dev)
    sg.kv4_plan(p, e, e, torch.empty(0, 4, dtype=torch.int32, device=dev))
    assert p.cu.tolist() == [0] and p.slots.tolist() == [-1] * 3 and p.info.tolist() == [0, 8, 0, 0]
    p = sg.Kv4Plan(2, 0, 16, 8, device=dev)
    t = torch.full((2, 2), -1, dtype=torch.int32, device=dev)
    sg.kv4_plan(p, ints([5, 0], dev), ints([0, 0], dev), t)
    assert p.cu.tolist() == [0, 0, 0] and p.seq.tolist() == [5, 0]


# ---- append and read ----------------------------------------------------------------------------

def fill_nan(cache):
    cache.data.fill_(0xFF)  # every scale and minimum a NaN until it is written


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,heads,page", [(64, 1, 16), (128, 3, 64), (256, 2, 32)])
def test_append_then_read(dev, dtype, d, heads, page):
    g = torch.Generator().manual_seed(d + heads)
    for n in (1, 2, 37, 200):
        nb = (n + page - 1) // page + 2
        cache = sg.Kv4Cache(nb, heads, d, page, device=dev)
        fill_nan(cache)
        before = cache.data.clone()
        slots = torch.randperm(nb * page, generator=g)[:n].int()
        x = torch.randn(n, 2 * heads + 1, d, generator=g)
        x[0, 0, :32] = 3.25                       # a group of equal values: scale 0
        x[-1, heads, 32:64] = 0.0
        x[0, 0, 32:64] *= 1e-6                    # a scale below f16's normal numbers
        x[n // 2, heads, :32] *= 2000.0
        x = x.to(dtype)
        xd = x.to(dev)
        sg.kv4_append(cache, xd[:, :heads], xd[:, heads:2 * heads], slots.to(dev))
        want = [U.quantized(x[:, :heads].float()), U.quantized(x[:, heads:2 * heads].float())]
        for out_type in TYPES:
            got = sg.kv4_read(cache, slots.to(dev), dtype=out_type)
            for a, b in zip(got, want):
                assert torch.equal(a.cpu(), b.float().to(out_type)), (n, out_type)
        # what is held: the code of a value is off by at most half a step, and the f16 minimum by half its unit
        v = x[:, :heads].double()
        r = v.unflatten(-1, (d // 32, 32))
        span = (r.amax(-1) - r.amin(-1))[..., None].expand(r.shape).flatten(-2)
        big = r.abs().amax(-1)[..., None].expand(r.shape).flatten(-2)
        assert ((want[0] - v).abs() <= span / 30 * (1 + 2 * U16) + 16 * U16 * span / 15 + 2 * U16 * big + 16 * 2.0 ** -24).all()
        # nothing else was touched
        free = torch.ones(nb * page, dtype=torch.bool)
        free[slots.long()] = False
        other = free.nonzero().flatten()[:64].int().to(dev)
        assert all(torch.isnan(t.float()).all() for t in sg.kv4_read(cache, other))
        assert (cache.data != before).sum() > 0 and cache.nonfinite.item() == 0


def test_append_odd_strides_match_aligned_ones(dev):
    d, heads, n = 128, 2, 19
    cache = [sg.Kv4Cache(2, heads, d, 16, device=dev) for _ in range(2)]
    slots = torch.arange(n, dtype=torch.int32, device=dev)
    for dtype in TYPES:
        flat = torch.randn(n * (2 * heads * d + 3) + 1, device=dev).to(dtype)
        x = flat[1:].view(n, -1)[:, :2 * heads * d].unflatten(1, (2 * heads, d))  # rows at odd elements
        y = x.contiguous()
        sg.kv4_append(cache[0], x[:, ::2], x[:, 1::2], slots)
        sg.kv4_append(cache[1], y[:, ::2].contiguous(), y[:, 1::2].contiguous(), slots)
        assert torch.equal(cache[0].data, cache[1].data)


def test_append_leaves_out_rows_without_a_slot(dev):
    cache = sg.Kv4Cache(3, 1, 64, 16, device=dev)
    k = torch.randn(4, 1, 64, device=dev)
    before = cache.data.clone()
    sg.kv4_append(cache, k, k, ints([-1, 48, 1 << 30, -(1 << 31)], dev))
    assert torch.equal(cache.data, before)
    sg.kv4_append(cache, k[:0], k[:0], ints([], dev))
    got = sg.kv4_read(cache, ints([-1, 48, 1 << 30], dev))
    assert all((t == 0).all() for t in got)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_infinities_and_nan(dev, dtype):
    d = 64
    x = torch.randn(6, 1, d)
    inf, nan = float("inf"), float("nan")
    x[0, 0, 3], x[1, 0, 4], x[2, 0, 5] = inf, -inf, nan
    x[3, 0, :32] = nan
    x[4, 0, :32], x[4, 0, 32:] = inf, -inf
    if dtype != torch.float16:
        x[5, 0, 7], x[5, 0, 40] = 1e30, -1e30
    x = x.to(dtype)
    cache = sg.Kv4Cache(1, 1, d, 16, device=dev)
    slots = torch.arange(6, dtype=torch.int32, device=dev)
    sg.kv4_append(cache, x.to(dev), x.to(dev), slots)
    k, v = sg.kv4_read(cache, slots, dtype=torch.float32)
    want = U.quantized(x.float()).float()
    assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want) and torch.isfinite(k).all()
    assert cache.nonfinite.item() == 2 * 6


# ---- attention ----------------------------------------------------------------------------------

def case(dev, lens, news, heads, d, page, seed, holes=0.0, extra_width=0, missing=()):
    """A cache that holds lens[i] positions of each request in blocks in a random
    order, everything else NaN."""
    g = torch.Generator(device=dev).manual_seed(seed)
    n = len(lens)
    width = max(1, max((x + page - 1) // page for x in lens)) + extra_width
    used = [(x + page - 1) // page for x in lens]
    nb = sum(used) + 3
    cache = sg.Kv4Cache(nb, heads, d, page, device=dev)
    fill_nan(cache)
    perm = torch.randperm(nb, generator=g, device=dev).tolist()
    tables = torch.full((n, width), -1, dtype=torch.int32)
    at = 0
    for i, u in enumerate(used):
        tables[i, :u] = torch.tensor(perm[at:at + u], dtype=torch.int32)
        at += u
    for i, length in enumerate(lens):
        if length:
            pos = torch.arange(length)
            slots = (tables[i][pos // page] * page + pos % page).int().to(dev)
            k = torch.randn(length, heads, d, device=dev, generator=g)
            sg.kv4_append(cache, k * 1.5, torch.randn(length, heads, d, device=dev, generator=g) + 0.3, slots)
    full = tables.clone()
    for i, j in missing:
        tables[i, j] = -1
    cu = [0]
    for x in news:
        cu.append(cu[-1] + x)
    return cache, tables.to(dev), full, ints(cu, dev), ints(lens, dev), g


def check(dev, cache, tables, full, cu, seq, q, scale, window, out, lse):
    d, page = cache.head_dim, cache.page
    cus, lens = cu.tolist(), seq.tolist()
    for i, length in enumerate(lens):
        a, b = cus[i], cus[i + 1]
        if a == b:
            continue
        pos = torch.arange(length)
        slots = (full[i][pos // page] * page + pos % page).int().to(dev)
        k, v = (t.double() for t in sg.kv4_read(cache, slots, dtype=torch.float32))
        seen = (tables[i].cpu()[pos // page] >= 0).to(dev)
        place = torch.arange(length - (b - a), length, device=dev)
        want, wlse, mag = U.attention(q[a:b].double(), k, v, place, seen, scale, window)
        # f32 everywhere: a score is a sum of D terms (D + 16 roundings of half a unit), and the weights carry
        # twice its error; the sums over positions another rounding each 2^-24 of sum p |v|, at most length of
        # them in a row.  16-bit types: the query is exact, weights and values may be rounded to f16 once
        # each, and the result to its type
        vmax = v.abs().max() if length else torch.zeros((), device=dev, dtype=torch.float64)
        eps = 2 * (d + 16) * U24 * mag + (length + 16) * U24
        err = eps[..., None] * vmax
        if q.dtype != torch.float32:
            err = err + 2 * U16 * vmax
        err = err + ROUND[q.dtype] * want.abs() + 1e-30
        got = out[a:b].double()
        assert torch.isfinite(got).all()
        assert ((got - want).abs() <= err).all(), (i, ((got - want).abs() / err).max().item())
        if lse is not None:
            gl = lse[a:b].double()
            none = torch.isinf(wlse)
            assert torch.equal(torch.isneginf(gl), none)
            assert ((gl - wlse).abs()[~none] <= (eps + 4 * U24 * wlse.abs())[~none]).all()
            assert (got[none] == 0).all()


SHAPES = [  # heads, group, D, page
    (1, 1, 64, 16), (2, 4, 64, 32), (4, 8, 128, 64), (8, 2, 128, 64), (1, 7, 128, 16), (2, 16, 128, 32), (1, 3, 256, 16),
    (2, 8, 256, 64), (1, 40, 64, 128)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group,d,page", SHAPES)
def test_attention_one_token(dev, dtype, heads, group, d, page):
    for k, lens in enumerate(([1], [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100], [700], [129, 0, 1, 4000, 64])):
        cache, tables, full, cu, seq, g = case(dev, lens, [1] * len(lens), heads, d, page, 10 * k + d)
        q = torch.randn(len(lens), heads * group, d, device=dev, generator=g).to(dtype)
        lse = torch.empty(len(lens), heads * group, device=dev)
        scale = d ** -0.5
        out = sg.kv4_attention(cache, q, cu, seq, tables, lse=lse, max_new=1)
        check(dev, cache, tables, full, cu, seq, q, scale, 0, out, lse)
        # without the optional arguments the same bits
        assert torch.equal(sg.kv4_attention(cache, q, cu, seq, tables, scale=scale), out)
    sg.device_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group,d,page", SHAPES)
def test_attention_several_tokens(dev, dtype, heads, group, d, page):
    # verify batches and prompt chunks, causal, ragged; also more new tokens than positions held (rows that see nothing)
    for k, (lens, news) in enumerate([([9, 40, 300], [9, 2, 9]), ([17], [17]), ([200, 1, 5, 0, 77], [130, 1, 9, 4, 0]),
                                      ([1000, 513], [65, 200])]):
        cache, tables, full, cu, seq, g = case(dev, lens, news, heads, d, page, 100 + k, extra_width=1)
        q = torch.randn(sum(news), heads * group, d, device=dev, generator=g).to(dtype)
        lse = torch.empty(sum(news), heads * group, device=dev)
        out = sg.kv4_attention(cache, q, cu, seq, tables, lse=lse, max_new=max(news))
        check(dev, cache, tables, full, cu, seq, q, d ** -0.5, 0, out, lse)
    sg.device_status()


@pytest.mark.parametrize("window", [1, 7, 64, 100, 100000])
@pytest.mark.parametrize("news", [[1, 1, 1], [70, 3, 300]])
def test_attention_window_and_missing_blocks(dev, window, news):
    heads, group, d, page = 2, 4, 128, 16
    lens = [400, 90, 333]
    for dtype in TYPES:
        missing = [(0, 3), (0, 24), (1, 0), (1, 1), (1, 2), (1, 3), (1, 4), (1, 5), (2, 20)]
        cache, tables, full, cu, seq, g = case(dev, lens, news, heads, d, page, window, missing=missing)
        q = torch.randn(sum(news), heads * group, d, device=dev, generator=g).to(dtype)
        lse = torch.empty(sum(news), heads * group, device=dev)
        out = sg.kv4_attention(cache, q, cu, seq, tables, window=window, scale=0.2, lse=lse, max_new=max(news))
        check(dev, cache, tables, full, cu, seq, q, 0.2, window, out, lse)


def test_attention_long_context(dev):
    # a long row spread over the whole device, next to short ones
    for dtype, heads, group, d in [(torch.float32, 2, 4, 128), (torch.bfloat16, 1, 8, 256), (torch.float16, 4, 1, 64)]:
        lens, news = [70001, 3, 9000], [1, 1, 1]
        cache, tables, full, cu, seq, g = case(dev, lens, news, heads, d, 64, 5)
        q = torch.randn(3, heads * group, d, device=dev, generator=g).to(dtype)
        lse = torch.empty(3, heads * group, device=dev)
        scratch = sg.kv4_attention_scratch(dev)
        out = sg.kv4_attention(cache, q, cu, seq, tables, lse=lse, max_new=1, scratch=scratch)
        check(dev, cache, tables, full, cu, seq, q, d ** -0.5, 0, out, lse)
        for _ in range(3):  # the scratch is ready for the next call, and the result does not depend on arrival order
            assert torch.equal(sg.kv4_attention(cache, q, cu, seq, tables, max_new=1, scratch=scratch), out)


def test_attention_strides_and_padding_tokens(dev):
    heads, group, d, page = 2, 4, 128, 64
    hq = heads * group
    for dtype in TYPES:
        lens, news = [300, 77], [5, 1]
        cache, tables, full, cu, seq, g = case(dev, lens, news, heads, d, page, 9, extra_width=2)
        n = sum(news) + 3                                              # three tokens of no request
        qkv = torch.randn(n, hq + 2 * heads, d, device=dev, generator=g).to(dtype)
        q = qkv[:, :hq]
        o = torch.full((hq, n, d + 1), 7.0, dtype=dtype, device=dev)   # heads first, odd rows
        lse = torch.empty(n, hq, device=dev)
        got = sg.kv4_attention(cache, q, cu, seq, tables, lse=lse, out=o.transpose(0, 1)[..., :d])
        check(dev, cache, tables, full, cu, seq, q, d ** -0.5, 0, got, lse)
        assert (got[sum(news):] == 0).all() and torch.isneginf(lse[sum(news):]).all()
        assert (o[..., d] == 7.0).all()
        odd = torch.empty(n * hq * d + 1, dtype=dtype, device=dev)[1:].view(n, hq, d).copy_(q)  # not 16-byte aligned
        assert torch.equal(sg.kv4_attention(cache, odd, cu, seq, tables), got)


def test_attention_extreme_queries_and_values(dev):
    # large, tiny and zero queries; values over f16's whole range in one cache
    heads, group, d, page = 1, 8, 128, 16
    for dtype in TYPES:
        cache = sg.Kv4Cache(8, heads, d, page, device=dev)
        fill_nan(cache)
        n = 100
        g = torch.Generator(device=dev).manual_seed(3)
        slots = torch.arange(n, dtype=torch.int32, device=dev)
        k = torch.randn(n, heads, d, device=dev, generator=g)
        v = torch.randn(n, heads, d, device=dev, generator=g)
        v[:, :, :32] *= 1e-5
        v[:, :, 32:64] *= 10.0
        v[50:, :, 32:64] *= 1000.0     # larger values come later
        tables = torch.arange(8, dtype=torch.int32, device=dev)[None]
        sg.kv4_append(cache, k, v, slots)
        q = torch.randn(1, group, d, device=dev, generator=g)
        q[0, 0] = 0
        q[0, 1] *= 1e-4
        q[0, 2] *= 200.0
        q[0, 3, 5] = 3000.0
        q = q.to(dtype)
        cu, seq = ints([0, 1], dev), ints([n], dev)
        lse = torch.empty(1, group, device=dev)
        out = sg.kv4_attention(cache, q, cu, seq, tables, lse=lse, max_new=1)
        kk, vv = (t.double() for t in sg.kv4_read(cache, slots, dtype=torch.float32))
        want, wl, mag = U.attention(q.double(), kk, vv, torch.tensor([n - 1], device=dev), torch.ones(n, dtype=torch.bool, device=dev),
                                    d ** -0.5, 0)
        for a in range(0, d, 32):     # by groups of channels: each by its own largest value
            vmax = vv[..., a:a + 32].abs().max()
            err = (2 * (d + 16) * U24 * mag + (n + 16) * U24)[..., None] * vmax + ROUND[dtype] * want[..., a:a + 32].abs()
            err = err + (2 * U16 * vmax if dtype != torch.float32 else 0) + 2.0 ** -25
            bad = ((out[..., a:a + 32].double() - want[..., a:a + 32]).abs() / err).max().item()
            assert bad <= 1, (dtype, a, bad)
        assert ((lse - wl).abs() <= 2 * (d + 16) * U24 * mag + 4 * U24 * wl.abs() + 16 * U24).all()


def test_attention_nan_query_stays_in_its_row(dev):
    heads, group, d, page = 1, 4, 64, 16
    for dtype in TYPES:
        cache, tables, full, cu, seq, g = case(dev, [50, 20], [3, 1], heads, d, page, 2)
        q = torch.randn(4, group, d, device=dev, generator=g).to(dtype)
        want = sg.kv4_attention(cache, q, cu, seq, tables)
        q[1, 2, 7] = float("nan")
        got = sg.kv4_attention(cache, q, cu, seq, tables)
        assert torch.isnan(got[1, 2]).all()
        got[1, 2] = want[1, 2]
        assert torch.equal(got, want)


def test_step_on_a_side_stream_and_in_a_graph(dev):
    # plan, append, attend on a stream of their own, then captured and replayed over growing lengths
    heads, group, d, page, n, width = 2, 2, 64, 16, 3, 8
    side = torch.cuda.Stream()
    cache = sg.Kv4Cache(n * width, heads, d, page, device=dev)
    plan = sg.Kv4Plan(n, n, page, n * width, device=dev)
    ring = torch.arange(n * width, dtype=torch.int32, device=dev)
    cursor = ints([0, n * width], dev)
    tables = torch.full((n, width), -1, dtype=torch.int32, device=dev)
    ctx, new = ints([0] * n, dev), ints([1] * n, dev)
    k, v = torch.empty(n, heads, d, device=dev), torch.empty(n, heads, d, device=dev)
    q, out = torch.empty(n, heads * group, d, device=dev), torch.empty(n, heads * group, d, device=dev)
    scratch = sg.kv4_attention_scratch(dev)
    torch.cuda.synchronize()

    def step():
        sg.kv4_plan(plan, ctx, new, tables, ring, cursor)
        sg.kv4_append(cache, k, v, plan.slots)
        sg.kv4_attention(cache, q, plan.cu, plan.seq, tables, max_new=1, out=out, scratch=scratch)
        cursor.copy_(plan.info[:2])
        ctx.copy_(plan.seq)

    g = torch.Generator(device=dev).manual_seed(1)
    ks, vs, graph = [], [], None
    for t in range(40):
        kk, vv, qq = (torch.randn(n, h, d, device=dev, generator=g) for h in (heads, heads, heads * group))
        ks.append(kk), vs.append(vv)
        k.copy_(kk), v.copy_(vv), q.copy_(qq)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            if t == 2:
                graph = torch.cuda.CUDAGraph()
                plan._turn = 0
                with torch.cuda.graph(graph, stream=side):
                    step()
            if graph is None:
                step()
            else:
                graph.replay()
        torch.cuda.synchronize()
        kq = U.quantized(torch.stack(ks).cpu()).to(dev)
        vq = U.quantized(torch.stack(vs).cpu()).to(dev)
        for i in range(n):
            want, _, mag = U.attention(qq[i:i + 1].double(), kq[:, i], vq[:, i], torch.tensor([t], device=dev),
                                       torch.ones(t + 1, dtype=torch.bool, device=dev), d ** -0.5, 0)
            err = (2 * (d + 16) * U24 * mag + (t + 17) * U24)[..., None] * vq.abs().max() + U24 * want.abs()
            assert ((out[i:i + 1].double() - want).abs() <= err).all(), (t, i)
    del graph


def test_refusals(dev):
    cache = sg.Kv4Cache(4, 2, 64, 16, device=dev)
    q = torch.zeros(1, 4, 64, device=dev)
    cu, seq, tables = ints([0, 1], dev), ints([1], dev), ints([[0]], dev)
    with pytest.raises(ValueError):
        sg.kv4_attention(cache, torch.zeros(1, 4, 128, device=dev), cu, seq, tables)
    with pytest.raises(sg.SgError):
        sg.kv4_attention(cache, torch.zeros(1, 3, 64, device=dev), cu, seq, tables)   # 3 query heads on 2
    with pytest.raises(TypeError):
        sg.kv4_attention(cache, q.double(), cu, seq, tables)
    with pytest.raises(TypeError):
        sg.kv4_attention(cache, q, cu.long(), seq, tables)
    with pytest.raises(ValueError):
        sg.kv4_attention(cache, q, cu, seq, tables.t().expand(1, 1).long())
    with pytest.raises(sg.SgError):
        sg.kv4_attention(cache, q, cu, seq, tables, scale=float("nan"))
    with pytest.raises(sg.SgError):
        sg.kv4_attention(cache, q, cu, seq, tables, scratch=torch.zeros(64, dtype=torch.uint8, device=dev))
    with pytest.raises(ValueError):
        sg.kv4_append(cache, torch.zeros(1, 1, 64, device=dev), torch.zeros(1, 1, 64, device=dev), ints([0], dev))
    with pytest.raises(ValueError):
        sg.kv4_append(cache, torch.zeros(1, 2, 64, device=dev), torch.zeros(1, 2, 64, device=dev).half(), ints([0], dev))
    with pytest.raises(ValueError):
        sg.kv4_append(cache, torch.zeros(2, 2, 64, device=dev), torch.zeros(2, 2, 64, device=dev), ints([0], dev))
    for bad in ((4, 2, 96, 16), (4, 2, 64, 24), (4, 2, 64, 8), (1 << 27, 1, 64, 16), (0, 1, 64, 16), (4, 0, 64, 16)):
        with pytest.raises(sg.SgError):
            sg.Kv4Cache(*bad, device=dev)
    with pytest.raises(ValueError):
        sg.Kv4Cache(4, 2, 64, 16, data=torch.zeros(16, dtype=torch.uint8, device=dev))
    p = sg.Kv4Plan(2, 4, 16, 4, device=dev)
    z = ints([0, 0], dev)
    with pytest.raises(ValueError):
        sg.kv4_plan(p, z[:1], z[:1], ints([[0]], dev))
    with pytest.raises(ValueError):
        sg.kv4_plan(p, z, z, torch.zeros(2, 2, device=dev))
    with pytest.raises(ValueError):
        sg.kv4_plan(p, z, z, torch.zeros(2, 2, dtype=torch.int32, device=dev), ring=p.ring)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,group,d,page", [(4, 8, 64, 16), (4, 8, 128, 64), (4, 8, 256, 16), (2, 7, 128, 32), (1, 16, 64, 128)])
@pytest.mark.parametrize("window", [0, 1, 50, 300])
def test_attention_many_rows(dev, dtype, heads, group, d, page, window):
    # enough rows for the tensor-core kernel: chunks against a context and without one, a request without new
    # tokens, rows that see nothing (no positions held, more new tokens than positions), blocks that are missing
    lens, news = [700, 300, 0, 40, 129, 65], [260, 300, 5, 60, 0, 1]
    assert sum(news) * heads * group * 7 > 26000
    missing = [(0, 0), (0, 2)] if page < 128 else [(0, 1)]
    cache, tables, full, cu, seq, g = case(dev, lens, news, heads, d, page, window + d, extra_width=1, missing=missing)
    n = sum(news) + 2                                                   # two tokens of no request
    q = torch.randn(n, heads * group, d, device=dev, generator=g).to(dtype)
    lse = torch.empty(n, heads * group, device=dev)
    out = sg.kv4_attention(cache, q, cu, seq, tables, window=window, lse=lse, max_new=300)
    check(dev, cache, tables, full, cu, seq, q, d ** -0.5, window, out, lse)
    assert (out[sum(news):] == 0).all() and torch.isneginf(lse[sum(news):]).all()
    assert torch.equal(sg.kv4_attention(cache, q, cu, seq, tables, window=window), out)
    sg.device_status()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_many_rows_strides_and_scales(dev, dtype):
    heads, group, d, page = 2, 4, 128, 16
    lens, news = [600, 513], [500, 513]
    cache, tables, full, cu, seq, g = case(dev, lens, news, heads, d, page, 77)
    n, hq = sum(news), heads * group
    qkv = torch.randn(n, hq + 2 * heads, d, device=dev, generator=g)
    qkv[3, 1] *= 1e-4
    qkv[4, 2] = 0
    qkv[5, 3] *= 100.0
    qkv = qkv.to(dtype)
    for scale in (d ** -0.5, -0.03):
        o = torch.full((hq, n, d + 1), 7.0, dtype=dtype, device=dev)    # heads first, odd rows
        lse = torch.empty(n, hq, device=dev)
        got = sg.kv4_attention(cache, qkv[:, :hq], cu, seq, tables, scale=scale, lse=lse, out=o.transpose(0, 1)[..., :d])
        check(dev, cache, tables, full, cu, seq, qkv[:, :hq], scale, 0, got, lse)
        assert (o[..., d] == 7.0).all()
        odd = torch.empty(n * hq * d + 1, dtype=dtype, device=dev)[1:].view(n, hq, d).copy_(qkv[:, :hq])
        assert torch.equal(sg.kv4_attention(cache, odd, cu, seq, tables, scale=scale), got)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_many_requests(dev, dtype):
    # more requests than one launch of the streaming kernel takes, of no and of a few tokens; and many short chunks
    g = torch.Generator().manual_seed(1)
    for n_req, most in [(2100, 1), (60, 24)]:
        lens = torch.randint(0, 40, (n_req,), generator=g).tolist()
        news = [min(x, int(torch.randint(0, most + 1, (1,), generator=g))) for x in lens]
        heads, group, d, page = 1, 4, 64, 16
        cache, tables, full, cu, seq, gg = case(dev, lens, news, heads, d, page, n_req)
        q = torch.randn(sum(news), heads * group, d, device=dev, generator=gg).to(dtype)
        lse = torch.empty(sum(news), heads * group, device=dev)
        out = sg.kv4_attention(cache, q, cu, seq, tables, lse=lse, max_new=most)
        for i in range(0, n_req, 97 if most == 1 else 7):               # some of them
            a, b = cu[i].item(), cu[i + 1].item()
            if a < b:
                check(dev, cache, tables[i:i + 1], full[i:i + 1], ints([0, b - a], dev), seq[i:i + 1], q[a:b], d ** -0.5, 0, out[a:b], lse[a:b])


def test_scratch_of_one_stream_serves_every_kernel(dev):
    # calls of different shapes one after another on one scratch
    scratch = sg.kv4_attention_scratch(dev)
    for k in range(3):
        for dtype, heads, group, d, lens, news in [(torch.float32, 2, 4, 128, [3000], [1]), (torch.float16, 1, 8, 256, [5000, 3], [2, 3]),
                                                   (torch.bfloat16, 4, 8, 64, [400], [300])]:
            cache, tables, full, cu, seq, g = case(dev, lens, news, heads, d, 32, k)
            q = torch.randn(sum(news), heads * group, d, device=dev, generator=g).to(dtype)
            lse = torch.empty(sum(news), heads * group, device=dev)
            out = sg.kv4_attention(cache, q, cu, seq, tables, lse=lse, scratch=scratch)
            check(dev, cache, tables, full, cu, seq, q, d ** -0.5, 0, out, lse)
