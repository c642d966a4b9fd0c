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
