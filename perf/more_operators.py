"""Microscaled 4-bit matrices and experts' products on them: what is measured of them.

Each case is one pass of one operator as a serving loop calls it.  `own` false: the plain form, elementary torch
operations in 32 bits.  `own` true: the calls of spindle_b200.  `exact` is the same from the definition in 64 bits.

A microscaled matrix holds 32 values along a row as c * 2^s: one exponent s (8 bits, s + 127) and 32 codes c of 4 bits, sign
and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  s is the exponent of the largest magnitude, after rounding it up to the next power
of two from 1.75 times a power on, less 2; codes are rounded to nearest, ties to the even code.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
MX = 17.0 / 32.0  # bytes a value


# ---- the cases ----------------------------------------------------------------------------------

def listed():
    return [
        # a verify batch's activations, as the decoder has them, to 4 bits and back
        dict(name="quantize-step", op="quantize", rows=9, cols=4096, dtype="f32"),
        # a long prompt's
        dict(name="quantize-prompt", op="quantize", rows=8191, cols=4096, dtype="bf16"),
        # one decoded token through a feed-forward matrix: latency and the weights' bytes
        dict(name="matmul-one", op="matmul", rows=1, cols=4096, out=14336, dtype="f32"),
        # a batch of decoding requests, the matrix back
        dict(name="matmul-batch", op="matmul", rows=33, cols=14336, out=4096, dtype="bf16"),
        # a whole prompt
        dict(name="matmul-prompt", op="matmul", rows=4096, cols=4096, out=14336, dtype="bf16"),
        # the choice of experts and the sorting of one decode step (128 experts, 8 a token)
        dict(name="route-step", op="route", tokens=16, experts=128, used=8, norm=True, masked=0.0, dtype="f32"),
        # of a long prompt
        dict(name="route-prompt", op="route", tokens=8191, experts=128, used=8, norm=True, masked=0.02, dtype="f32"),
        # gate and up of one decode step: 16 tokens' experts
        dict(name="experts-step", op="experts", part="up", tokens=16, dim=2048, ff=768, experts=128, used=8, dtype="f32"),
        # of a prompt
        dict(name="experts-prompt", op="experts", part="up", tokens=4096, dim=2048, ff=768, experts=128, used=8, dtype="bf16"),
        # and the way back down of an odd one
        dict(name="experts-down", op="experts", part="down", tokens=4095, dim=2048, ff=768, experts=128, used=8, dtype="bf16"),
        # the experts' results of one decode step put together
        dict(name="combine-step", op="combine", tokens=16, dim=2048, experts=128, used=8, masked=0.0, dtype="f32"),
        # of a long prompt
        dict(name="combine-prompt", op="combine", tokens=8191, dim=2048, experts=128, used=8, masked=0.02, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "matmul", "matmul", "matmul", "route", "experts", "experts", "experts", "combine"])
    c = dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]))
    if op == "quantize":
        c["cols"] = 32 * _log(rng, 2, 512)
        c["rows"] = _log(rng, 1, 8191 * 4096 // c["cols"])
    elif op == "matmul":
        c["cols"], c["out"] = 32 * _log(rng, 4, 512), _log(rng, 100, 20000)
        c["out"] = min(c["out"], 58000000 // c["cols"])
        c["rows"] = _log(rng, 1, min(8192, 200000000000 // (c["cols"] * c["out"])))
    else:
        c["experts"], c["used"] = rng.choice([8, 32, 60, 64, 128, 256]), rng.choice([1, 2, 4, 6, 8])
        if op == "route":
            c.update(tokens=_log(rng, 1, 8191), norm=rng.random() < 0.7, masked=rng.choice([0.0, 0.02, 0.3]))
        elif op == "combine":
            c.update(dim=8 * _log(rng, 32, 512), masked=rng.choice([0.0, 0.02, 0.3]))
            c["tokens"] = _log(rng, 1, 8191 * 8 * 2048 // (c["used"] * c["dim"]))
        else:
            c.update(part=rng.choice(["up", "down"]), dim=32 * _log(rng, 8, 128), ff=32 * _log(rng, 8, 64))
            c["ff"] = max(32, min(c["ff"], 200000000 // (c["experts"] * c["dim"]) // 32 * 32))
            c["tokens"] = _log(rng, 1, min(4096, 51000000000 // (c["used"] * c["dim"] * c["ff"])))
    return c


# ---- what a program has in hand -----------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"quantize": _prepare_quantize, "matmul": _prepare_matmul, "route": _prepare_route, "experts": _prepare_experts,
         "combine": _prepare_combine}[case["op"]](case, g)
    s["case"] = case
    dt = DTYPES[case["dtype"]]
    if own:
        # the handles that a serving loop makes once: weights laid out, the plan of the experts, its buffers
        import spindle_b200 as sg
        if "weights" in s:
            w = [sg.mx4_quantize(_values(c, e)) for c, e in s.pop("weights")]
            s["w"], s["up"] = w[0], w[1] if len(w) == 2 else None
        if case["op"] == "quantize":
            s["m"] = sg.Mx4(case["rows"], case["cols"], device="cuda")
            s["out"] = torch.empty(case["rows"], case["cols"], dtype=dt, device="cuda")
        elif case["op"] == "matmul":
            s["out"] = torch.empty(case["rows"], case["out"], dtype=dt, device="cuda")
            s["scratch"] = sg.mx4_scratch(s["w"], case["rows"])
        else:
            s["plan"] = sg.MoePlan(case["tokens"], case["used"], case["experts"], device="cuda")
            if case["op"] != "route":
                sg.moe_sort(s["ids"], s["weight"], s["plan"])
            if case["op"] == "experts":
                s["out"] = torch.empty(case["tokens"] * case["used"], s["w"].rows, dtype=dt, device="cuda")
                s["scratch"] = sg.mx4_scratch(s["w"], s["plan"])
            elif case["op"] == "combine":
                s["out"] = torch.empty(case["tokens"], case["dim"], dtype=dt, device="cuda")
    return s


def _activations(g, rows, cols):
    """Rows as a norm leaves them, a few channels stronger than the others, as models have them."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    return x * (1 + 7 * (torch.rand(cols, device="cuda", generator=g) < 0.02))


def _weights(g, *shape):
    """Codes and exponents of a matrix of the size of its rows' inverse root."""
    return _plain_codes(torch.randn(*shape, device="cuda", generator=g) * shape[-1] ** -0.5)


def _prepare_quantize(case, g):
    return dict(x=_activations(g, case["rows"], case["cols"]).to(DTYPES[case["dtype"]]))


def _prepare_matmul(case, g):
    return dict(x=_activations(g, case["rows"], case["cols"]).to(DTYPES[case["dtype"]]), weights=[_weights(g, case["out"], case["cols"])])


def _logits(case, g):
    """A router's logits, some experts more liked than others, some of them closed to a token."""
    x = torch.randn(case["tokens"], case["experts"], device="cuda", generator=g) * 1.5 + torch.randn(case["experts"], device="cuda", generator=g) * 0.5
    if case.get("masked"):
        x.masked_fill_(torch.rand(x.shape, device="cuda", generator=g) < case["masked"], float("-inf"))
    return x


def _prepare_route(case, g):
    return dict(logits=_logits(case, g).to(DTYPES[case["dtype"]]))


def _chosen(case, g):
    ids, weight = _plain_choice(_logits(case, g), case["used"], True)
    return dict(ids=ids, weight=weight, **{k: v for k, v in zip(("first", "order", "place"), _plain_sort(ids, case["experts"]))})


def _prepare_experts(case, g):
    s = _chosen(case, g)
    n, dim, ff, e = case["tokens"], case["dim"], case["ff"], case["experts"]
    if case["part"] == "up":
        s["x"], s["weights"] = _activations(g, n, dim), [_weights(g, e, ff, dim), _weights(g, e, ff, dim)]
    else:
        s["x"] = _activations(g, n * case["used"], ff) * torch.rand(n * case["used"], ff, device="cuda", generator=g)
        s["weights"] = [_weights(g, e, dim, ff)]
    s["x"] = s["x"].to(DTYPES[case["dtype"]])
    s["most"] = int((s["first"][1:] - s["first"][:-1]).max())
    return s


def _prepare_combine(case, g):
    s = _chosen(case, g)
    s["y"] = torch.randn(case["tokens"] * case["used"], case["dim"], device="cuda", generator=g).to(DTYPES[case["dtype"]])
    return s


# ---- one pass -------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"quantize": _plain_quantize, "matmul": _plain_matmul, "route": _plain_route, "experts": _plain_experts,
                "combine": _plain_combine}[op](s)
    import spindle_b200 as sg
    if op == "quantize":
        return sg.mx4_dequantize(sg.mx4_quantize(s["x"], out=s["m"]), out=s["out"])
    if op == "matmul":
        return sg.mx4_matmul(s["x"], s["w"], out=s["out"], scratch=s["scratch"])
    if op == "route":
        p = sg.moe_route(s["logits"], s["plan"], norm=c["norm"])
        return {"ids": p.ids, "weights": p.weights, "first": p.first, "order": p.order, "place": p.place}
    if op == "experts":
        return sg.mx4_experts(s["x"], s["w"], s["plan"], up=s["up"], out=s["out"], scratch=s["scratch"])
    return sg.moe_combine(s["y"], s["plan"], out=s["out"])


# ---- the plain forms ------------------------------------------------------------------------------

def _plain_codes(x):
    """Codes (uint8, one a value) and exponents (uint8, one for 32 values) of the rows of x."""
    x = x.float().unflatten(-1, (x.shape[-1] // 32, 32))
    top = x.abs().amax(-1).view(torch.int32)
    e = ((top + 0x200000) >> 23).sub_(2).clamp_(min=0)
    bad = top >= 0x7F800000                                    # an infinity or a NaN among the 32: no numbers
    y = torch.ldexp(x, (127 - e)[..., None])
    a = y.abs()
    c = (a > 0.25).to(torch.uint8)
    for limit, even in ((0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)):
        c += (a >= limit) if even else (a > limit)
    c += (y < 0) * torch.tensor(8, dtype=torch.uint8, device=x.device)
    return torch.where(bad[..., None], 0, c).flatten(-2), torch.where(bad, 255, e).to(torch.uint8)


def _values(codes, e):
    """What codes and exponents stand for, in f32."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = table[codes.int()].unflatten(-1, (codes.shape[-1] // 32, 32))
    v = torch.ldexp(v, e.int()[..., None] - 127)
    return torch.where(e[..., None] == 255, float("nan"), v).flatten(-2)


def _plain_quantize(s):
    return _values(*_plain_codes(s["x"])).to(s["x"].dtype)


def _plain_matmul(s):
    x = _values(*_plain_codes(s["x"]))
    return (x @ _values(*s["weights"][0]).T).to(s["x"].dtype)


def _plain_choice(logits, used, norm):
    """The used likeliest experts of each token, equal ones by rising number, and their weights; -1: none left."""
    x = logits.float()
    value, ids = torch.sort(x, dim=1, descending=True, stable=True)
    value, ids = value[:, :used], ids[:, :used]
    if value.shape[1] < used:
        fill = (0, used - value.shape[1])
        value, ids = torch.nn.functional.pad(value, fill, value=float("-inf")), torch.nn.functional.pad(ids, fill)
    none = value == float("-inf")
    top = torch.where(none[:, :1], 0.0, value[:, :1])
    e = (value - top).exp()
    total = e.sum(1, keepdim=True) if norm else (x - top).exp().sum(1, keepdim=True)
    return torch.where(none, -1, ids).int(), torch.where(none, 0.0, e / total)


def _plain_sort(ids, experts):
    """First sorted place of each expert, each place's pair (token * used + choice) and each pair's place; -1: none."""
    flat = ids.flatten().long()
    key, order = torch.sort(torch.where(flat < 0, experts, flat), stable=True)
    first = torch.searchsorted(key, torch.arange(experts + 1, device=ids.device))
    at = torch.arange(len(flat), device=ids.device)
    there = at < first[-1]
    place = torch.empty_like(at)
    place[order] = torch.where(there, at, -1)
    return first.int(), torch.where(there, order, -1).int(), place.view(ids.shape).int()


def _plain_route(s):
    c = s["case"]
    ids, weight = _plain_choice(s["logits"], c["used"], c["norm"])
    first, order, place = _plain_sort(ids, c["experts"])
    return {"ids": ids, "weights": weight, "first": first, "order": order, "place": place}


def _plain_experts(s):
    c = s["case"]
    x = _values(*_plain_codes(s["x"]))
    count = s["first"][1:] - s["first"][:-1]
    j = torch.arange(s["most"], device=x.device)
    at = (s["first"][:-1, None] + j).long()
    here = j < count[:, None]                                   # [experts, most]
    row = s["order"][at.clamp(max=len(s["order"]) - 1)].long()
    source = x[row // c["used"] if c["part"] == "up" else at.clamp(max=len(x) - 1)]
    y = [torch.bmm(source, _values(*w).transpose(1, 2)) for w in s["weights"]]
    y = y[0] / (1 + (-y[0]).exp()) * y[1] if len(y) == 2 else y[0]
    out = torch.zeros(len(s["order"]), y.shape[-1], dtype=s["x"].dtype, device=x.device)
    out[at[here]] = y[here].to(out.dtype)
    return out


def _plain_combine(s):
    place = s["place"].long()
    y = s["y"][place.clamp(min=0)].float()
    w = torch.where(place < 0, 0.0, s["weight"])
    return (torch.where(place[..., None] < 0, 0.0, y) * w[..., None]).sum(1).to(s["y"].dtype)


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    op, es = case["op"], SIZES[case["dtype"]]
    if op == "quantize":
        values = case["rows"] * case["cols"]
        return {"bytes": values * (2.0 * es + 2 * MX), "flops": 4.0 * values}
    if op == "matmul":
        m, k, n = case["rows"], case["cols"], case["out"]
        return {"bytes": n * k * MX + m * (k + n) * float(es), "flops": 2.0 * m * n * k}
    pairs = case["tokens"] * case["used"]
    if op == "route":
        return {"bytes": case["tokens"] * case["experts"] * float(es) + 16.0 * pairs + 4.0 * case["experts"], "flops": 3.0 * case["tokens"] * case["experts"]}
    if op == "combine":
        return {"bytes": (pairs + case["tokens"]) * float(case["dim"] * es) + 8.0 * pairs, "flops": 2.0 * pairs * case["dim"]}
    up = case["part"] == "up"
    # the experts that tokens of equal chances reach
    reached = case["experts"] * (1 - (1 - min(1.0, case["used"] / case["experts"])) ** case["tokens"])
    weights = case["dim"] * case["ff"] * (2 if up else 1)
    rows_in, rows_out = (case["tokens"] * case["dim"], pairs * case["ff"]) if up else (pairs * case["ff"], pairs * case["dim"])
    return {"bytes": reached * weights * MX + (rows_in + rows_out) * float(es) + 8.0 * pairs, "flops": 2.0 * pairs * weights}


# ---- the definition in 64 bits --------------------------------------------------------------------

def exact(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "quantize":
        return _exact_rounded(_prepare_quantize(case, g)["x"])
    if op == "matmul":
        s = _prepare_matmul(case, g)
        w = _exact_values(*s["weights"][0])
        return torch.cat([_exact_rounded(x) @ w.T for x in s["x"].split(1024)])
    if op == "route":
        x = _prepare_route(case, g)["logits"].double()
        best = x.topk(min(case["used"], x.shape[1]), 1).values
        best = torch.nn.functional.pad(best, (0, case["used"] - best.shape[1]), value=float("-inf"))
        p = best - torch.logsumexp(best if case["norm"] else x, 1, keepdim=True)
        p = torch.where(torch.isneginf(best), 0.0, p.exp())
        return {"ids": None, "weights": p, "first": None, "order": None, "place": None}
    if op == "experts":
        return _exact_experts(case, _prepare_experts(case, g))
    s = _prepare_combine(case, g)
    out = torch.zeros(case["tokens"], case["dim"], dtype=torch.float64, device="cuda")
    pair = torch.arange(case["tokens"] * case["used"], device="cuda")[s["place"].flatten() >= 0]
    for some in pair.split(1 << 14):
        y = s["y"][s["place"].flatten()[some].long()].double() * s["weight"].flatten()[some].double()[:, None]
        out.index_add_(0, some // case["used"], y)
    return out


def _exact_rounded(x):
    """What 4 bits hold of the rows of x: the nearest of the numbers that there are, by searching among them."""
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    top = b.abs().max(-1, keepdim=True).values
    two = torch.floor(torch.log2(top.clamp(min=2.0 ** -149)) + 1e-13)
    two = torch.where(top >= 1.75 * torch.pow(2.0, two), two + 1, two)
    step = torch.pow(torch.full_like(two, 2.0), (two - 2).clamp(min=-127))
    there = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 6], dtype=torch.float64, device=x.device)
    z = (b.abs() / step).clamp(max=6)
    low = torch.searchsorted(there[:8].contiguous(), z, right=True) - 1
    below, above = there[low], there[low + 1]
    up = (z - below > above - z) | ((z - below == above - z) & (low % 2 == 1))
    return (torch.where(up, above, below) * step * b.sign()).reshape(x.shape)


def _exact_values(codes, e):
    c = codes.long()
    size, sign = c % 8, 1.0 - 2.0 * (c // 8).double()
    # half steps up to 2, then one more bit of exponent: 2 3 4 6
    v = torch.where(size < 4, size.double() / 2, torch.where(size % 2 == 0, 1.0, 1.5) * torch.where(size < 6, 2.0, 4.0))
    return (sign * v * torch.pow(torch.tensor(2.0, dtype=torch.float64, device=c.device), e.double() - 127).repeat_interleave(32, -1))


def _exact_experts(case, s):
    at = s["first"].tolist()
    out = None
    for e in range(case["experts"]):
        if at[e] == at[e + 1]:
            continue
        rows = torch.arange(at[e], at[e + 1], device="cuda")
        if case["part"] == "up":
            rows = torch.div(s["order"][at[e]:at[e + 1]].long(), case["used"], rounding_mode="floor")
        x = _exact_rounded(s["x"][rows])
        y = [x @ _exact_values(c[e], k[e]).T for c, k in s["weights"]]
        y = y[0] * torch.sigmoid(y[0]) * y[1] if len(y) == 2 else y[0]
        if out is None:
            out = torch.zeros(len(s["order"]), y.shape[1], dtype=torch.float64, device="cuda")
        out[at[e]:at[e + 1]] = y
    return out
