"""The paged 4-bit KV cache and token log probabilities: what is measured of them.

Each case is one pass of one operator as a serving loop calls it.  `own` false: the plain form, elementary torch
operations in 32 bits.  `own` true: the calls of spindle_b200.  `exact` is the same from the definition in 64 bits.

A cache block holds `page` positions; for one KV head a block is page / 16 tiles of 20 * D bytes (D = head_dim, G = D / 32
groups of 32 values, each with an f16 scale s and minimum m, a value being m + s * c for a code c of 0..15):
  K codes [16 positions][D / 2], V codes [8 position pairs][D], then f16 K scales [8][G][2], K minima [16][G],
  V scales [8][G][2], V minima [8][G][2] (the last index of [8][G][2] is the position inside its pair).
  K: 32-bit word ((g // 4) * 4 + j) * 4 + g % 4 (D = 64: j * 2 + g) of a position holds d = 32 g + 8 j + n in nibble n.
  V: 32-bit word ((g // 4) * 8 + j) * 4 + g % 4 (D = 64: j * 2 + g) of a pair holds d = 32 g + 4 j + n in nibble n of its
  low half for the even position and of its high half for the odd one.
"""
import math

import torch

own = False

F16_MAX = 65504.0
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases ----------------------------------------------------------------------------------

def listed():
    return [
        # a decode step's bookkeeping: 64 requests of one new token each, now and then one that ends
        dict(name="plan-decode", op="plan", n_req=64, ctx=4096, new=1, page=64),
        # prompts admitted together with running requests: a million slots, ragged
        dict(name="plan-prompts", op="plan", n_req=509, ctx=8191, new=4096, page=16),
        # the K/V rows of one decode step of 32 requests enter the cache
        dict(name="append-decode", op="append", tokens=32, heads=8, dim=128, page=64, dtype="f16"),
        # a long prompt's rows enter the cache
        dict(name="append-prompt", op="append", tokens=24001, heads=8, dim=128, page=64, dtype="bf16"),
        # one chat at a short context: latency (16 query and 8 KV heads of 128, the dense 0.6B shape)
        dict(name="attend-one", op="attend", n_req=1, ctx=1037, new=1, heads=8, group=2, dim=128, page=64, window=0, dtype="f16"),
        # a batch of decoding requests of different lengths (32 query and 4 KV heads, the 30B-A3B shape)
        dict(name="attend-batch", op="attend", n_req=64, ctx=8192, new=1, heads=4, group=8, dim=128, page=64, window=0, dtype="bf16"),
        # one request over a very long context
        dict(name="attend-long", op="attend", n_req=1, ctx=131071, new=1, heads=8, group=4, dim=128, page=32, window=0, dtype="f16"),
        # speculative verify batches of 9 tokens, in f32 as the decoder's activations are
        dict(name="attend-verify", op="attend", n_req=16, ctx=2050, new=9, heads=8, group=2, dim=128, page=64, window=0, dtype="f32"),
        # two prompt chunks against the context before them
        dict(name="attend-prompt", op="attend", n_req=2, ctx=8100, new=1024, heads=4, group=8, dim=128, page=64, window=0, dtype="bf16"),
        # the probabilities of one decoded token
        dict(name="logprobs-one", op="logprobs", rows=1, vocab=151936, top=5, dtype="f32", few=0.0),
        # a batch of decoding requests, some constrained by a grammar to a few tokens
        dict(name="logprobs-batch", op="logprobs", rows=65, vocab=151936, top=20, dtype="f32", few=0.1),
        # the log probabilities of a whole prompt, a vocabulary of odd size
        dict(name="logprobs-prompt", op="logprobs", rows=2048, vocab=151935, top=1, dtype="bf16", few=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "logprobs", "logprobs"])
    if op == "plan":
        c = dict(op=op, n_req=_log(rng, 1, 512), ctx=_log(rng, 1, 8191), new=_log(rng, 1, 4096), page=rng.choice([16, 32, 64, 128]))
    elif op == "append":
        c = dict(op=op, heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128, 256]), page=rng.choice([16, 32, 64]),
                 dtype=rng.choice(["f32", "f16", "bf16"]))
        c["tokens"] = _log(rng, 1, 12000000 // (c["heads"] * c["dim"]))
    elif op == "attend":
        dim, heads, group = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8, 16])
        c = dict(op=op, heads=heads, group=group, dim=dim, page=rng.choice([16, 32, 64, 128]),
                 window=rng.choice([0, 0, 0, 511, 1024]), dtype=rng.choice(["f32", "f16", "f16", "bf16", "bf16"]))
        kind = rng.choice(["decode", "decode", "verify", "prompt"])
        c["new"] = 1 if kind == "decode" else _log(rng, 2, 16) if kind == "verify" else _log(rng, 17, 1024)
        most = 200000000 // (heads * dim)                      # cached values of the whole batch
        c["ctx"] = max(c["new"], _log(rng, 17, min(131072, most) if kind == "decode" else min(8192, most)))
        fit = min(most, 400000000 // (c["new"] * heads * group)) // c["ctx"]   # and its scores
        c["n_req"] = _log(rng, 1, max(1, min(256, fit)))
    else:
        c = dict(op=op, vocab=_log(rng, 1000, 200000), top=rng.choice([0, 1, 5, 20, 20, 64]), dtype=rng.choice(["f32", "f16", "bf16"]),
                 few=rng.choice([0.0, 0.0, 0.1, 0.5]))
        c["rows"] = _log(rng, 1, max(1, min(4096, 300000000 // c["vocab"])))
    return c


def _lengths(case):
    """Cached and new positions of each request: the first has the most of both, the others fewer and fewer."""
    n, ctx, new = case["n_req"], case["ctx"], case["new"]
    news = [max(1, new - i * new // (2 * n)) for i in range(n)]
    return [max(news[i], ctx - i * ctx * 3 // (4 * n)) for i in range(n)], news


# ---- what a program has in hand -----------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"plan": _prepare_plan, "append": _prepare_append, "attend": _prepare_attend, "logprobs": _prepare_logprobs}[case["op"]](case, g)
    s["case"] = case
    if own:
        # the handles that a serving loop makes once: the cache's description, its output buffers and scratch
        import spindle_b200 as sg
        if "data" in s:
            s["cache"] = sg.Kv4Cache(s["n_blocks"], case["heads"], case["dim"], case["page"], data=s["data"])
        if case["op"] == "plan":
            s["handle"] = sg.Kv4Plan(case["n_req"], s["max_tokens"], case["page"], s["n_blocks"], device="cuda")
        elif case["op"] == "append":
            s["out"] = tuple(torch.empty(case["tokens"], case["heads"], case["dim"], dtype=torch.float16, device="cuda") for _ in range(2))
        elif case["op"] == "attend":
            s["out"] = torch.empty_like(s["q"])
            s["lse"] = torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda")
            s["scratch"] = sg.kv4_attention_scratch(device="cuda")
        else:
            s["out"] = sg.LogProbs(case["rows"], case["top"], device="cuda")
    return s


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _prepare_plan(case, g):
    lens, news = _lengths(case)
    n, page = case["n_req"], case["page"]
    ctx = torch.tensor([a - b for a, b in zip(lens, news)], device="cuda")
    # the lengths before this step differ from seed to seed, at most the case's; about one request in 32 ends here
    ctx = ctx - (torch.rand(n, device="cuda", generator=g) * ctx.clamp(max=page)).long()
    new = torch.tensor(news, device="cuda")
    new = torch.where(torch.rand(n, device="cuda", generator=g) < 1 / 32, -1, new)
    width = (max(lens) + page - 1) // page + 1
    n_blocks = n * width
    perm = torch.randperm(n_blocks, device="cuda", generator=g).int()
    have = (ctx + page - 1) // page
    own_block = torch.arange(width, device="cuda") < have[:, None]
    tables = torch.where(own_block, perm.view(n, width), -1).int()
    # the free blocks lie in a ring from `head` to `tail`
    free = perm.view(n, width)[~own_block]
    head = int(torch.randint(n_blocks, (1,), device="cuda", generator=g))
    ring = torch.full((n_blocks,), -1, dtype=torch.int32, device="cuda")
    ring[(head + torch.arange(len(free), device="cuda")) % n_blocks] = free
    return dict(ctx=ctx.int(), new=new.int(), tables=tables, ring=ring, cursor=_ints([head, head + len(free)]),
                max_tokens=sum(news), n_blocks=n_blocks)


def _prepare_append(case, g):
    t, h, d, page = case["tokens"], case["heads"], case["dim"], case["page"]
    # K and V as the two parts of one projection's output; K has a few strong channels, as models have
    kv = torch.randn(t, 2, h, d, device="cuda", generator=g)
    kv[:, 0] *= 1 + 4 * (torch.rand(h, d, device="cuda", generator=g) < 0.03)
    kv = kv.to(DTYPES[case["dtype"]])
    blocks = (t + page - 1) // page + 8
    table = torch.randperm(blocks, device="cuda", generator=g)
    pos = torch.arange(t, device="cuda") + int(torch.randint(page, (1,), device="cuda", generator=g))
    slots = (table[pos // page] * page + pos % page).int()
    data = torch.zeros(blocks * h * (page // 16) * 20 * d, dtype=torch.uint8, device="cuda")
    return dict(k=kv[:, 0], v=kv[:, 1], slots=slots, data=data, n_blocks=blocks)


def _prepare_attend(case, g):
    lens, news = _lengths(case)
    n, h, d, page = case["n_req"], case["heads"], case["dim"], case["page"]
    width = (max(lens) + page - 1) // page
    used = [(x + page - 1) // page for x in lens]
    blocks = sum(used)
    perm = torch.randperm(blocks, device="cuda", generator=g).int()
    use = torch.tensor(used, device="cuda")
    row = torch.arange(width, device="cuda") + (torch.cumsum(use, 0) - use)[:, None]
    tables = torch.where(torch.arange(width, device="cuda") < use[:, None], perm[row.clamp(max=blocks - 1)], -1).int()
    data = torch.zeros(blocks * h * (page // 16) * 20 * d, dtype=torch.uint8, device="cuda")
    # every block filled with quantized rows, a piece at a time
    strong = 1 + 4 * (torch.rand(h, d, device="cuda", generator=g) < 0.03)
    step = max(1, (1 << 26) // (h * d))
    for at in range(0, blocks * page, step):
        slots = torch.arange(at, min(blocks * page, at + step), device="cuda")
        k = torch.randn(len(slots), h, d, device="cuda", generator=g) * strong
        v = torch.randn(len(slots), h, d, device="cuda", generator=g)
        _plain_append(data, k, v, slots, h, d, page)
    cu = [0]
    for x in news:
        cu.append(cu[-1] + x)
    q = torch.randn(cu[-1], h * case["group"], d, device="cuda", generator=g).to(DTYPES[case["dtype"]])
    return dict(q=q, cu=_ints(cu), seq=_ints(lens), tables=tables, data=data, n_blocks=blocks, max_new=max(news),
                scale=1 / math.sqrt(d))


def _prepare_logprobs(case, g):
    n, v = case["rows"], case["vocab"]
    x = torch.randn(n, v, device="cuda", generator=g) * 2.5
    # some likely tokens in each row, at places of their own
    x.scatter_add_(1, torch.randint(v, (n, 8), device="cuda", generator=g), 9 * torch.rand(n, 8, device="cuda", generator=g))
    if case["few"]:
        allowed = torch.randint(v, (n, 40), device="cuda", generator=g)
        mask = torch.ones(n, v, dtype=torch.bool, device="cuda").scatter_(1, allowed, False)
        mask &= (torch.rand(n, 1, device="cuda", generator=g) < case["few"])
        x.masked_fill_(mask, float("-inf"))
    # half of the given tokens are the likeliest, as a decoder picks them, the others any allowed one
    x = x.to(DTYPES[case["dtype"]])
    best = x.argmax(1)
    other = torch.randint(v, (n,), device="cuda", generator=g)
    at = torch.arange(n, device="cuda")
    pick = (torch.rand(n, device="cuda", generator=g) < 0.5) | torch.isinf(x[at, other])
    return dict(logits=x, tokens=torch.where(pick, best, other).int())


# ---- one pass -------------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if not own:
        return {"plan": _plain_plan, "append": _plain_append_run, "attend": _plain_attend, "logprobs": _plain_logprobs}[op](s)
    import spindle_b200 as sg
    if op == "plan":
        p = sg.kv4_plan(s["handle"], s["ctx"], s["new"], s["tables"], s["ring"], s["cursor"])
        return {"cu": p.cu, "seq": p.seq, "pos": p.pos, "slots": p.slots, "info": p.info, "tables": s["tables"], "ring": s["ring"]}
    if op == "append":
        sg.kv4_append(s["cache"], s["k"], s["v"], s["slots"])
        k, v = sg.kv4_read(s["cache"], s["slots"], out=s["out"])
        return {"k": k, "v": v, "data": s["data"]}
    if op == "attend":
        o = sg.kv4_attention(s["cache"], s["q"], s["cu"], s["seq"], s["tables"], scale=s["scale"], window=s["case"]["window"],
                             max_new=s["max_new"], out=s["out"], lse=s["lse"], scratch=s["scratch"])
        return {"out": o, "lse": s["lse"]}
    p = sg.logprobs(s["logits"], s["tokens"], top=s["case"]["top"], out=s["out"])
    return _named(s["case"], p.logprob, p.entropy, p.rank, p.top_ids, p.top_logprobs)


def _named(case, logprob, entropy, rank, ids, tops):
    got = {"logprob": logprob, "entropy": entropy, "rank": rank}
    return {**got, "top_ids": ids, "top_logprobs": tops} if case["top"] else got


# ---- the plain forms ------------------------------------------------------------------------------

def _plain_plan(s):
    page, n_blocks, most = s["case"]["page"], s["n_blocks"], s["max_tokens"]
    ctx, new, tables, ring = s["ctx"].long(), s["new"].long(), s["tables"], s["ring"]
    head, tail = s["cursor"][0].long(), s["cursor"][1].long()
    come, ends = new.clamp(min=0), new < 0
    have, need = (ctx + page - 1) // page, (ctx + come + page - 1) // page
    want = torch.where(ends, 0, need - have)
    first = torch.cumsum(want, 0) - want
    cu = torch.nn.functional.pad(torch.cumsum(come, 0), (1, 0))
    # blocks for the new positions
    width = tables.shape[1]
    j = torch.arange(width, device=ctx.device)
    rank = first[:, None] + j - have[:, None]
    block = torch.where(rank < tail - head, ring[((head + rank) % n_blocks)], -1)
    grown = torch.where((j >= have[:, None]) & (j < need[:, None]) & ~ends[:, None], block, tables)
    # the blocks of the requests that end go back
    back = torch.where(ends, have, 0)
    at = (torch.cumsum(back, 0) - back)[:, None] + j
    freed = ends[:, None] & (j < have[:, None])
    ring[((tail + at) % n_blocks)[freed]] = tables[freed]
    tables.copy_(grown)
    # each new position's request, position and slot
    t = torch.arange(most, device=ctx.device)
    r = torch.searchsorted(cu[1:], t, right=True).clamp(max=len(ctx) - 1)
    here = t < cu[-1]
    pos = torch.where(here, ctx[r] + t - cu[r], -1)
    b = grown[r, (pos // page).clamp(min=0)].long()
    slots = torch.where(here & (b >= 0), b * page + pos % page, -1)
    taken = torch.minimum(want.sum(), tail - head)
    turn = (head + taken) // n_blocks * n_blocks  # the head stays inside the ring
    info = torch.stack([head + taken - turn, tail + back.sum() - turn, cu[-1], want.sum() - taken])
    seq = torch.where(ends, 0, ctx + come)
    return {"cu": cu.int(), "seq": seq.int(), "pos": pos.int(), "slots": slots.int(), "info": info.int(), "tables": tables, "ring": ring}


def _plain_quantize(x, d):
    """Codes [.., D], scales and minima [.., G] of the rows of x, all in f32 (the latter rounded to f16)."""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=F16_MAX, neginf=-F16_MAX).clamp(-F16_MAX, F16_MAX)
    x = x.unflatten(-1, (d // 32, 32))
    m = (x.amin(-1) + 0.0).half().float()
    s = ((x.amax(-1) - m).clamp(min=0) * (1.0 / 15.0)).half().float()
    r = torch.where(s > 0, 1.0 / s, 0.0)
    c = torch.round(((x - m[..., None]) * r[..., None]).clamp(0, 15))
    return c.flatten(-2).to(torch.int32), s, m


def _views(data, h, d, page):
    """The parts of the cache: K codes, V codes (int16), K scales, K minima, V scales, V minima, all [blocks, heads, tiles, ..]."""
    g = d // 32
    b = data.view(-1, h, page // 16, 20 * d)
    w, f = b.view(torch.int16), b.view(torch.float16)
    kc = b[..., :8 * d].unflatten(-1, (16, d // 2))
    vc = w[..., 4 * d:8 * d].unflatten(-1, (8, d // 4, 2))
    p = f[..., 8 * d:].unflatten(-1, (4, d // 2))
    pair = [p[..., i, :].unflatten(-1, (8, g, 2)) for i in (0, 2, 3)]
    return kc, vc, pair[0], p[..., 1, :].unflatten(-1, (16, g)), pair[1], pair[2]


def _plain_append(data, k, v, slots, h, d, page):
    g = d // 32
    gg = min(g, 4)
    ok = slots >= 0
    k, v, slots = k[ok], v[ok], slots[ok].long()
    kq, ks, km = _plain_quantize(k, d)
    vq, vs, vm = _plain_quantize(v, d)
    # K: nibbles to bytes, then the words of 4 bytes into their order
    n = kq.unflatten(-1, (g // gg, gg, 4, 4, 2))
    kb = (n[..., 0] | n[..., 1] << 4).to(torch.uint8).movedim(-2, -3).flatten(-4)
    # V: 4 nibbles to a half word, which lies in the low or the high half of its word by the position
    n = vq.unflatten(-1, (g // gg, gg, 8, 4))
    vb = (n[..., 0] | n[..., 1] << 4 | n[..., 2] << 8 | n[..., 3] << 12)
    vb = torch.where(vb > 32767, vb - 65536, vb).to(torch.int16).transpose(-1, -2).flatten(-3)
    blk, pos = slots // page, slots % page
    tile, row = pos // 16, pos % 16
    pair, side = row // 2, row % 2
    kc, vc, kss, kms, vss, vms = _views(data, h, d, page)
    kc[blk, :, tile, row] = kb
    vc[blk, :, tile, pair, :, side] = vb
    kss[blk, :, tile, pair, :, side] = ks.half()
    kms[blk, :, tile, row] = km.half()
    vss[blk, :, tile, pair, :, side] = vs.half()
    vms[blk, :, tile, pair, :, side] = vm.half()


def _plain_values(kc, vc, ks, km, vs, vm, d):
    """K and V in f32, [.., D], of gathered rows: kc [.., D / 2] bytes, vc [.., D / 4] int16, the others [.., G]."""
    g = d // 32
    gg = min(g, 4)
    n = kc.to(torch.int32).unflatten(-1, (g // gg, 4, gg, 4)).movedim(-3, -2)
    kq = torch.stack([n & 15, n >> 4], -1).flatten(-5).float()
    n = vc.to(torch.int32).unflatten(-1, (g // gg, 8, gg)).transpose(-1, -2)
    vq = torch.stack([n & 15, n >> 4 & 15, n >> 8 & 15, n >> 12 & 15], -1).flatten(-4).float()
    out = []
    for c, s, m in ((kq, ks, km), (vq, vs, vm)):
        out.append((m.float()[..., None] + s.float()[..., None] * c.unflatten(-1, (g, 32))).flatten(-2))
    return out


def _plain_append_run(s):
    c = s["case"]
    h, d, page = c["heads"], c["dim"], c["page"]
    _plain_append(s["data"], s["k"], s["v"], s["slots"], h, d, page)
    slots = s["slots"].long()
    blk, pos = slots // page, slots % page
    tile, row = pos // 16, pos % 16
    pair, side = row // 2, row % 2
    kc, vc, ks, km, vs, vm = _views(s["data"], h, d, page)
    k, v = _plain_values(kc[blk, :, tile, row], vc[blk, :, tile, pair, :, side], ks[blk, :, tile, pair, :, side],
                         km[blk, :, tile, row], vs[blk, :, tile, pair, :, side], vm[blk, :, tile, pair, :, side], d)
    return {"k": k.half(), "v": v.half(), "data": s["data"]}


def _plain_attend(s):
    c = s["case"]
    h, d, page, group, window = c["heads"], c["dim"], c["page"], c["group"], c["window"]
    q, cu, seq, tables = s["q"], s["cu"].long(), s["seq"].long(), s["tables"]
    n, width = tables.shape
    rows = [x[tables.clamp(min=0).long()].transpose(2, 1) for x in _views(s["data"], h, d, page)]  # [n, heads, blocks, tiles, ..]
    kc, vc, ks, km, vs, vm = rows
    vc, ks, vs, vm = (x.transpose(-1, -2).flatten(-3, -2) for x in (vc, ks, vs, vm))  # pairs to positions
    kc, vc, ks, km, vs, vm = (x.flatten(2, 4) for x in (kc, vc, ks, km, vs, vm))
    k, v = _plain_values(kc, vc, ks, km, vs, vm, d)              # [n, heads, positions, D]
    del rows, kc, vc
    # the new tokens of each request, as rows of (token, head of the group)
    most = s["max_new"]
    j = torch.arange(most, device=q.device)
    count = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + j).clamp(max=len(q) - 1)
    qf = q.float()[at].view(n, most, h, group, d).permute(0, 2, 1, 3, 4).reshape(n, h, most * group, d)
    score = (qf @ k.transpose(-1, -2)).mul_(s["scale"])          # [n, heads, rows, positions]
    t = torch.arange(width * page, device=q.device)
    place = seq[:, None] - count[:, None] + j                    # [n, most]
    see = (t <= place[..., None]) & (t < seq[:, None, None])
    if window:
        see &= t > place[..., None] - window
    see &= (tables >= 0).repeat_interleave(page, 1)[:, None]
    see = see[:, None, :, None].expand(n, 1, most, group, -1).flatten(2, 3)
    score.masked_fill_(~see, float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()).squeeze(-1)
    # back to packed tokens
    r = torch.searchsorted(cu[1:], torch.arange(len(q), device=q.device), right=True)
    i = torch.arange(len(q), device=q.device) - cu[r]
    o = o.view(n, h, most, group, d)[r, :, i].reshape(len(q), h * group, d)
    return {"out": o.to(q.dtype), "lse": lse.view(n, h, most, group)[r, :, i].reshape(len(q), h * group)}


def _plain_logprobs(s):
    x, tok = s["logits"].float(), s["tokens"].long()
    top = s["case"]["top"]
    m = x.amax(1, keepdim=True)
    dist = x - m
    e = dist.exp()
    z = e.sum(1, keepdim=True)
    entropy = z.log() - torch.where(e > 0, e * dist, 0.0).sum(1, keepdim=True) / z
    given = x.gather(1, tok[:, None])
    logprob = given - m - z.log()
    ahead = (x > given) | ((x == given) & (torch.arange(x.shape[1], device=x.device) < tok[:, None]))
    rank = ahead.sum(1)
    ids = tops = None
    if top:
        value, order = torch.sort(x, dim=1, descending=True, stable=True)
        ids, tops = order[:, :top].int().contiguous(), value[:, :top] - m - z.log()
    return _named(s["case"], logprob.squeeze(1), entropy.squeeze(1), rank.int(), ids, tops)


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "plan":
        lens, news = _lengths(case)
        blocks = sum((a + case["page"] - 1) // case["page"] for a in lens)
        return {"bytes": 16.0 * case["n_req"] + 8.0 * sum(news) + 8.0 * blocks, "flops": 0.0}
    if op == "append":
        values = 2.0 * case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": values * (SIZES[case["dtype"]] + 2 * 5 / 8 + 2), "flops": 6 * values}
    if op == "attend":
        lens, news = _lengths(case)
        hq, d, window = case["heads"] * case["group"], case["dim"], case["window"] or 1 << 60
        read = sum(min(a, window + b - 1) for a, b in zip(lens, news))
        pairs = sum(min(a - b + 1 + i, window) for a, b in zip(lens, news) for i in range(b))
        return {"bytes": read * case["heads"] * d * 2 * 5 / 8 + sum(news) * hq * (2 * d * SIZES[case["dtype"]] + 4),
                "flops": 4.0 * pairs * hq * d}
    n, v, top = case["rows"], case["vocab"], case["top"]
    return {"bytes": n * (v * SIZES[case["dtype"]] + 16.0 + 8 * top), "flops": 5.0 * n * v}


# ---- the definition in 64 bits --------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers only
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "append":
        s = _prepare_append(case, g)
        return {"k": _exact_rounded(s["k"]), "v": _exact_rounded(s["v"]), "data": None}
    if case["op"] == "attend":
        return _exact_attend(case, _prepare_attend(case, g))
    return _exact_logprobs(case, _prepare_logprobs(case, g))


def _exact_rounded(x):
    """What the cache holds for the rows of x."""
    t, h, d = x.shape
    x = x.double().reshape(t, h, d // 32, 32)
    low = x.min(-1, keepdim=True).values.to(torch.float16).double()
    step = ((x.max(-1, keepdim=True).values - low) / 15).clamp(min=0).to(torch.float16).double()
    code = ((x - low) / step.masked_fill(step == 0, 1.0)).clamp(0, 15).round()
    return (low + step * code).reshape(t, h, d)


def _exact_rows(case, data, slots, head):
    """K and V [positions, D] of one head in 64 bits, value by value from the layout above."""
    d, page, h = case["dim"], case["page"], case["heads"]
    groups = d // 32
    tile = ((slots // page * h + head) * (page // 16) + slots % page // 16)[:, None] * (20 * d)
    t, e = (slots % 16)[:, None], torch.arange(d, device=slots.device)[None]
    g = e // 32

    def word(j, width):
        return (g // 4 * width + j) * 4 + g % 4 if groups > 2 else j * 2 + g

    n = e % 8
    kb = data[tile + t * (d // 2) + word(e % 32 // 8, 4) * 4 + n // 2].long()
    kq = torch.where(n % 2 == 1, kb >> 4, kb & 15).double()
    n = e % 4
    vb = data[tile + 8 * d + t // 2 * d + word(e % 32 // 4, 8) * 4 + t % 2 * 2 + n // 2].long()
    vq = torch.where(n % 2 == 1, vb >> 4, vb & 15).double()
    f = data.view(torch.float16)
    at = tile // 2 + 8 * d
    paired = (t // 2 * groups + g) * 2 + t % 2
    ks, km = f[at + paired].double(), f[at + d // 2 + t * groups + g].double()
    vs, vm = f[at + d + paired].double(), f[at + d + d // 2 + paired].double()
    return km + ks * kq, vm + vs * vq


def _exact_attend(case, s):
    lens, news = _lengths(case)
    group, page, window = case["group"], case["page"], case["window"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], float("-inf"), dtype=torch.float64, device="cuda")
    first = 0
    for i, (length, new) in enumerate(zip(lens, news)):
        t = torch.arange(length, device="cuda")
        slots = s["tables"][i].long()[t // page] * page + t % page
        place = torch.arange(length - new, length, device="cuda")[:, None]
        hidden = (t > place) | ((t <= place - window) if window else torch.zeros_like(t > place))
        for head in range(case["heads"]):
            k, v = _exact_rows(case, s["data"], slots, head)
            mine = slice(head * group, (head + 1) * group)
            q = s["q"][first:first + new, mine].double().transpose(0, 1)
            z = torch.matmul(q, k.T) * s["scale"]
            z = z.masked_fill(hidden, float("-inf"))
            all_ = torch.logsumexp(z, -1)
            out[first:first + new, mine] = torch.matmul(torch.exp(z - all_[..., None]), v).transpose(0, 1)
            lse[first:first + new, mine] = all_.T
        first += new
    return {"out": out, "lse": lse}


def _exact_logprobs(case, s):
    n = case["rows"]
    logprob, entropy, tops = [], [], []
    for at in range(0, n, 128):
        x = s["logits"][at:at + 128].double()
        lp = x - torch.logsumexp(x, 1, keepdim=True)
        logprob.append(lp[torch.arange(len(lp), device="cuda"), s["tokens"][at:at + 128].long()])
        entropy.append(-torch.special.xlogy(lp.exp(), lp.exp()).sum(1))
        if case["top"]:
            tops.append(lp.topk(case["top"], 1).values)
    return _named(case, torch.cat(logprob), torch.cat(entropy), None, None, torch.cat(tops) if tops else None)
