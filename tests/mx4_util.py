"""Plain 64-bit forms of the microscaled 4-bit matrix and expert operators, for their tests."""
import torch

# what a code's magnitude can be, and where the next one up begins to be nearer (a tie goes to the even code)
SIZES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def quantized(x):
    """The values that 4 bits hold of the rows of x [.., cols], in 64 bits, by the definition."""
    b = x.double().cpu().unflatten(-1, (x.shape[-1] // 32, 32))
    top = b.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)                       # top = m 2^e, m in [0.5, 1)
    s = torch.where(top > 0, e - 1 - 2 + (m >= 0.875), torch.full_like(e, -200)).clamp(min=-127)
    y = torch.ldexp(b.abs(), -s)
    dist = (y[..., None] - SIZES).abs()
    near = dist.amin(-1, keepdim=True)
    even = torch.where(dist == near, torch.arange(8) % 2, 9).argmin(-1)  # of two equally near ones the even one
    v = torch.ldexp(SIZES[even], s) * torch.where(b < 0, -1.0, 1.0).double()
    return torch.where(torch.isfinite(top), v, float("nan")).flatten(-2).to(x.device)


def half_step(t, dtype):
    """Bound of the rounding of values t to dtype (its smallest step at least)."""
    tiny = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[dtype]
    return t.abs() * (torch.finfo(dtype).eps / 2) + tiny


def product(xq, wq, uq=None):
    """x w^T (silu of it times x up^T) in 64 bits of quantized operands, and a bound of what sums in f32 may be off: the
    tensor cores add 64 products at a time and may cut a sum off, a unit in its last place (2^-23) each; one more for
    what is added at the end, of parts."""
    n = xq.shape[-1] // 64 + 10
    y, dy = xq @ wq.T, (xq.abs() @ wq.abs().T) * (n * 2.0 ** -23)
    if uq is None:
        return y, dy
    u, du = xq @ uq.T, (xq.abs() @ uq.abs().T) * (n * 2.0 ** -23)
    s = y * torch.sigmoid(y)
    # |silu'| is below 1.1; exponential, sum, quotient and product are off by less than 8 half steps of the result
    return s * u, 1.1 * dy * u.abs() + s.abs() * du + 1.1 * dy * du + (s * u).abs() * (8 * 2.0 ** -24) + 1e-37


def close(got, want, bound):
    """Whether got (of its type) is want within bound and its own rounding."""
    d = (got.double() - want).abs()
    return bool((d <= bound + half_step(want.abs() + bound, got.dtype)).all())


def choice(logits, k, norm, prune=0.0):
    """Ids and weights of each token, one by one."""
    ids, weights = [], []
    for row in logits.double().cpu().tolist():
        order = sorted((i for i in range(len(row)) if row[i] != float("-inf")), key=lambda i: (-row[i], i))[:k]
        x = torch.tensor([row[i] for i in order], dtype=torch.float64)
        top = x[0] if len(order) else 0.0
        p = torch.exp(x - top)
        keep = len(order)
        if prune > 0 and keep > 2:
            least = max(keep // 2, 2)
            if prune >= 1:
                keep = min(max(int(prune), least), keep)
            else:
                n, target = 0, float(p.sum()) * (1 - prune)
                while n < keep and (n < least or float(p[:n].sum()) < target):
                    n += 1
                keep = n
        total = p[:keep].sum() if norm else torch.exp(torch.tensor(row, dtype=torch.float64) - top).sum()
        ids.append(order[:keep] + [-1] * (k - keep))
        weights.append((p[:keep] / total).tolist() + [0.0] * (k - keep))
    return torch.tensor(ids, dtype=torch.int32).view(-1, k), torch.tensor(weights, dtype=torch.float64).view(-1, k)


def sort(ids, n_expert):
    """first, order and place of the pairs, by Python's stable sort."""
    flat = ids.flatten().tolist()
    pairs = sorted((p for p in range(len(flat)) if 0 <= flat[p] < n_expert), key=lambda p: flat[p])
    count = [0] * n_expert
    for p in pairs:
        count[flat[p]] += 1
    first = [0]
    for c in count:
        first.append(first[-1] + c)
    place = [-1] * len(flat)
    for s, p in enumerate(pairs):
        place[p] = s
    i = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return i(first), i(pairs + [-1] * (len(flat) - len(pairs))), i(place).view(ids.shape)
