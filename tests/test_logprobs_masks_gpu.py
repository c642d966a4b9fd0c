"""logprobs on the GPU where masks leave few tokens or hold large finite numbers, against
64 bits: the paths that fill up the alternatives, and the sums over masked stretches."""
import pytest
import torch

import spindle_b200 as sg

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = float("inf")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 151936), (40, 151936), (9, 2500), (700, 4099)])
def test_fewer_allowed_than_alternatives(dev, dtype, rows, vocab):
    # 0 to top - 1 tokens left in a row, in one CTA's stretch or spread over a cluster's: the rest of the alternatives
    # are minus infinities in rising id.  Every thread of a CTA has to take the same way here, whichever is first.
    top = 20
    g = torch.Generator(device=dev).manual_seed(rows)
    x = torch.full((rows, vocab), -INF, device=dev, dtype=dtype)
    want = []
    for r in range(rows):
        n = r % top
        at = torch.randperm(vocab if r % 2 else 600, generator=g, device=dev)[:n]
        x[r, at] = (torch.randperm(64, generator=g, device=dev)[:n] * 0.25).to(dtype)
        here = at[x[r, at].float().argsort(descending=True)].tolist()
        want.append((here + [i for i in range(2 * top) if i not in set(here)])[:top])
    want = torch.tensor(want, dtype=torch.int32)
    tokens = want[:, 3].to(dev).contiguous()
    rank = torch.full((rows,), 3, dtype=torch.int32)
    for _ in range(20):
        got = sg.logprobs(x, tokens, top=top)
        assert torch.equal(got.top_ids.cpu(), want) and torch.equal(got.rank.cpu(), rank)
    lp = x.double().log_softmax(1).gather(1, want.to(dev).long())
    lp[torch.isnan(lp)] = -INF                             # a row with nothing left
    fin = torch.isfinite(lp)
    assert torch.equal(torch.isneginf(got.top_logprobs), ~fin)
    # distances up to 16 (half a unit in the last place each), a sum of at most 20 terms, its logarithm
    assert ((got.top_logprobs.double() - lp).abs()[fin] <= (16 + 8 * 16 + 20) * 2.0 ** -24).all()


def finite_masks(dev, dtype, rows, vocab, mask, places):
    """Rows of one large finite number but for a few likely tokens in given places; in 64 bits the masked ones
    have probability 0.  Returns logits, tokens, and log probability, entropy and alternatives in 64 bits."""
    x = torch.full((rows, vocab), mask, device=dev, dtype=dtype)
    at = torch.tensor([(p + 37 * r) % vocab for r in range(rows) for p in places], device=dev).view(rows, -1)
    x.scatter_(1, at, (torch.arange(len(places), device=dev) * 0.5 - 1).to(dtype).expand(rows, -1))
    few = x.gather(1, at).double()
    lp = few.log_softmax(1)
    return x, at, lp, -(lp.exp() * lp).sum(1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 151936), (65, 151936), (900, 70001)])
@pytest.mark.parametrize("mask", ["lowest", -1e38, -1e37, -1e9])
def test_large_finite_masks(dev, dtype, rows, vocab, mask):
    # the allowed tokens come a thread's second turn or later: its sum moves from the mask's value to theirs
    low = float(torch.finfo(dtype).min)
    mask = low if mask == "lowest" else max(mask, low)
    places = [vocab - 5, vocab - 70, vocab - 3000, vocab // 2 + 9000, vocab - 9001]
    x, at, lp, ent = finite_masks(dev, dtype, rows, vocab, mask, places)
    got = sg.logprobs(x, at[:, 2].int().contiguous(), top=5)
    # values below 2 apart: a few units in the last place of 1 for distances, exponentials, five terms and the logarithm
    tol = (16 + 8 * 2 + 5) * 2.0 ** -24
    assert (got.entropy.double() - ent).abs().max() <= tol
    assert (got.logprob.double() - lp[:, 2]).abs().max() <= tol
    assert torch.equal(got.top_ids.long(), at.flip(1)) and (got.rank == 2).all()


@pytest.mark.parametrize("rows,vocab", [(1, 151936), (65, 151936), (900, 70001)])
@pytest.mark.parametrize("part", [0.7, 0.8])
def test_large_finite_masks_below_bf16s_lowest(dev, rows, vocab, part):
    # masks whose distance times log2 e is past f32's range, in a type that reads them sixteen values at a time
    places = [vocab - 5, vocab - 70, vocab - 3000, vocab // 2 + 9000, vocab - 9001]
    x, at, lp, ent = finite_masks(dev, torch.bfloat16, rows, vocab, part * torch.finfo(torch.bfloat16).min, places)
    x[:, ::7] = x[0, 0] * 0.9                                    # more than one of them
    x.scatter_(1, at, (torch.arange(5, device=dev) * 0.5 - 1).bfloat16().expand(rows, -1))
    got = sg.logprobs(x, at[:, 2].int().contiguous(), top=5)
    tol = (16 + 8 * 2 + 5) * 2.0 ** -24
    assert (got.entropy.double() - ent).abs().max() <= tol
    assert (got.logprob.double() - lp[:, 2]).abs().max() <= tol
    assert torch.equal(got.top_ids.long(), at.flip(1)) and (got.rank == 2).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_huge_logit_after_ordinary_ones(dev, dtype):
    vocab = 151936
    g = torch.Generator(device=dev).manual_seed(7)
    x = torch.randn(3, vocab, device=dev, generator=g).to(dtype)
    for r, at in enumerate((vocab - 9, vocab // 2, 100000)):
        x[r, at] = torch.finfo(dtype).max
    got = sg.logprobs(x, torch.tensor([vocab - 9, vocab // 2, 100000], dtype=torch.int32, device=dev), top=1)
    assert (got.entropy == 0).all() and (got.logprob == 0).all() and (got.rank == 0).all()
