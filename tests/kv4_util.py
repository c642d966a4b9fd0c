"""Plain 64-bit forms of the paged 4-bit cache operators, for their tests."""
import torch

F16_MAX = 65504.0


def quantized(x):
    """What the cache holds for the rows of x [.., D] (float32, on the CPU), in 64
    bits: the codes by the documented f32 steps, the values from the f16 parameters."""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=F16_MAX, neginf=-F16_MAX).clamp(-F16_MAX, F16_MAX)
    g = x.unflatten(-1, (x.shape[-1] // 32, 32))
    m = g.amin(-1, keepdim=True).half().float()
    s = ((g.amax(-1, keepdim=True) - m).clamp(min=0) * torch.tensor(1.0 / 15.0)).half().float()
    r = torch.where(s > 0, torch.tensor(1.0) / s, torch.zeros(()))
    c = torch.round(((g - m) * r).clamp(0, 15))
    return (m.double() + s.double() * c.double()).flatten(-2)


def attention(q, k, v, place, see_block, scale, window):
    """q [n, Hq, D], k and v [len, H, D] (64 bits), place [n]: each token's position,
    see_block [len] bool.  Returns out, lse and, per (token, head), the largest
    scale * sum |q k| that a seen position has."""
    n, hq, d = q.shape
    group = hq // k.shape[1]
    t = torch.arange(k.shape[0], device=q.device)
    see = (t <= place[:, None]) & see_block
    if window:
        see &= t > place[:, None] - window
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("nhd,thd->nht", q, kk) * scale
    mag = torch.einsum("nhd,thd->nht", q.abs(), kk.abs()) * abs(scale)
    s = s.masked_fill(~see[:, None], float("-inf"))
    mag = mag.masked_fill(~see[:, None], 0.0)
    none = ~see.any(1)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(none[:, None], torch.zeros_like(lse), lse)[..., None])
    out = torch.einsum("nht,thd->nhd", torch.where(see[:, None], p, torch.zeros_like(p)), vv)
    return out, lse, mag.amax(-1) if k.shape[0] else torch.zeros_like(lse)


def plan(ctx, new, tables, ring, head, tail, page, n_blocks, max_tokens):
    """kv4_plan in plain Python; tables and ring are lists that it updates."""
    cu, seq, pos, slots, missing = [0], [], [], [], 0
    taken, back = 0, 0
    free = tail - head
    for i, (c, a) in enumerate(zip(ctx, new)):
        have = (c + page - 1) // page
        if a < 0:
            for j in range(have):
                if tables[i][j] >= 0:
                    ring[(tail + back) % n_blocks] = tables[i][j]
                    back += 1
            cu.append(cu[-1])
            seq.append(0)
            continue
        for p in range(c, c + a):
            j = p // page
            if p % page == 0:
                if taken < free:
                    tables[i][j] = ring[(head + taken) % n_blocks]
                else:
                    tables[i][j] = -1
                    missing += 1
                taken += 1
            pos.append(p)
            slots.append(tables[i][j] * page + p % page if tables[i][j] >= 0 else -1)
        cu.append(cu[-1] + a)
        seq.append(c + a)
    pad = max_tokens - len(pos)
    h = head + min(taken, free)
    turn = h // n_blocks * n_blocks
    return cu, seq, pos + [-1] * pad, slots + [-1] * pad, [h - turn, tail + back - turn, cu[-1], missing]
