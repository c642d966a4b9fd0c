"""logprobs on the GPU against a plain form in 64 bits."""
import pytest
import torch

import spindle_b200 as sg

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
U24 = 2.0 ** -24


def reference(x, tokens, top):
    x = x.double().cpu()
    vocab = x.shape[1]
    none = torch.isneginf(x).all(1, keepdim=True)
    m = x.amax(1, keepdim=True)
    d = torch.where(none, torch.full_like(x, float("-inf")), x - m)
    e = d.exp()
    z = e.sum(1, keepdim=True)
    lp = torch.where(none, d, d - z.log())
    ent = torch.where(none[:, 0], torch.zeros(()).double(), (z.log() - torch.where(e > 0, e * d, torch.zeros(()).double()).sum(1, keepdim=True) / z)[:, 0])
    t = tokens.long().cpu()
    ok = (t >= 0) & (t < vocab)
    tt = t.clamp(0, vocab - 1)
    # NaN before everything, then falling, equal ones by index
    key = torch.where(torch.isnan(x), torch.full_like(x, float("inf")), x)
    isn = torch.isnan(x)
    order = torch.stack([torch.tensor(sorted(range(vocab), key=lambda i: (not isn[r, i], -key[r, i].item(), i))) for r in range(len(x))])
    rank = (order == tt[:, None]).int().argmax(1)
    given = lp.gather(1, tt[:, None])[:, 0]
    given[~ok] = float("nan")
    rank[~ok] = -1
    ids = order[:, :top]
    return given, ent, rank.int(), ids.int(), lp.gather(1, ids)


def close(got, want, x):
    # an f32 distance x - m (half a unit of the larger), e^d and the sum: a few units of the sum relative, ln z a few more
    g, w = got.double().cpu(), want
    assert torch.equal(torch.isnan(g), torch.isnan(w))
    fin = torch.isfinite(w)
    assert torch.equal(g[~fin & ~torch.isnan(w)], w[~fin & ~torch.isnan(w)])
    big = x.double().cpu().abs()
    big = torch.where(torch.isfinite(big), big, torch.zeros(()).double()).amax(1)
    tol = (16 + 8 * big + x.shape[1] ** 0.5) * U24
    tol = tol if g.dim() == 1 else tol[:, None].expand(g.shape)
    assert ((g - w).abs()[fin] <= (tol + 4 * U24 * w.abs())[fin]).all()


def check(x, tokens, top, out=None):
    got = sg.logprobs(x, tokens, top=top, out=out)
    torch.cuda.synchronize()
    lp, ent, rank, ids, tops = reference(x, tokens, top)
    assert got.rank.tolist() == rank.tolist()
    assert got.top_ids.tolist() == ids.tolist()
    close(got.logprob, lp, x)
    close(got.entropy, ent, x)
    close(got.top_logprobs, tops, x)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (2, 1, 0), (1, 2, 2), (3, 31, 5), (5, 64, 64), (2, 1000, 20), (7, 4097, 1),
                                            (1, 50257, 20), (3, 32000, 64), (1, 151936, 5)])
def test_random_rows(dev, dtype, rows, vocab, top):
    g = torch.Generator(device=dev).manual_seed(vocab + rows)
    x = (torch.randn(rows, vocab, device=dev, generator=g) * 3).to(dtype)
    tokens = torch.randint(vocab, (rows,), device=dev, generator=g).int()
    tokens[0] = x[0].float().argmax().int()
    check(x, tokens, top)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows(dev, dtype):
    # more rows than CTAs fit on the device, few enough values to check every one
    g = torch.Generator(device=dev).manual_seed(4)
    x = (torch.randn(700, 531, device=dev, generator=g) * 3).to(dtype)
    check(x, torch.randint(-1, 531, (700,), device=dev, generator=g).int(), 7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40, 5003, 33000])
def test_ties_go_to_the_lowest_id(dev, dtype, vocab):
    g = torch.Generator(device=dev).manual_seed(vocab)
    few = torch.randint(0, 3, (4, vocab), device=dev, generator=g).float()
    few[1] = 0.5                                      # all equal
    few[2] = 0.0
    few[2, vocab // 2:] = -0.0                        # the zeros are equal too
    few[3] = torch.arange(vocab, device=dev).div(10, rounding_mode="floor").neg()  # falling, in tens
    x = few.to(dtype)
    check(x, torch.tensor([vocab - 1, vocab // 3, vocab - 2, 25], dtype=torch.int32, device=dev), 20)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [300, 20011])
def test_masked_rows(dev, dtype, vocab):
    g = torch.Generator(device=dev).manual_seed(vocab)
    inf = float("inf")
    x = (torch.randn(7, vocab, device=dev, generator=g) * 2).to(dtype)
    x[0] = -inf                                        # nothing left
    x[1, :vocab - 3] = -inf                            # fewer left than alternatives are wanted
    x[2] = -inf
    x[2, 17] = 1.0                                     # one left: probability 1
    x[3] = torch.finfo(dtype).min                      # masked with the lowest value, all of it
    x[4, 5:] = torch.finfo(dtype).min
    x[5, ::2] = -inf
    x[6, 100] = torch.finfo(dtype).max                 # far above the rest
    tokens = torch.tensor([3, vocab - 2, 17, 9, 2, 4, 100], dtype=torch.int32, device=dev)
    got = check(x, tokens, 20)
    assert torch.isneginf(got.logprob[0]) and got.entropy[0] == 0
    assert got.logprob[2] == 0 and got.entropy[2] == 0 and got.rank[2] == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_and_infinity_in_a_row(dev, dtype):
    inf, nan = float("inf"), float("nan")
    for vocab in (200, 9001):
        g = torch.Generator(device=dev).manual_seed(1)
        x = torch.randn(5, vocab, device=dev, generator=g).to(dtype)
        x[0, 33] = nan
        x[1, 44] = inf
        x[2, 7] = nan
        x[2, 8] = inf
        x[2, 3] = nan
        x[3] = nan
        tokens = torch.tensor([33, 5, 8, 199, 2], dtype=torch.int32, device=dev)
        got = sg.logprobs(x, tokens, top=10)
        _, _, rank, ids, _ = reference(x, tokens, 10)
        assert got.top_ids.tolist() == ids.tolist() and got.rank.tolist() == rank.tolist()
        assert torch.isnan(got.logprob[:4]).all() and torch.isnan(got.entropy[:4]).all() and torch.isnan(got.top_logprobs[:4]).all()
        assert torch.isfinite(got.logprob[4]) and torch.isfinite(got.entropy[4])


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_alignment_and_kept_outputs(dev, dtype):
    rows, vocab = 6, 3001
    flat = torch.randn(rows * (vocab + 6) + 1, device=dev).to(dtype)
    x = flat[1:].view(rows, vocab + 6)[:, :vocab]     # rows at every alignment
    tokens = torch.arange(rows, dtype=torch.int32, device=dev) * 7 - 1
    out = sg.LogProbs(rows, 3, device=dev)
    assert check(x, tokens, 3, out=out) is out
    y = x.contiguous()
    again = sg.logprobs(y, tokens, top=3)
    assert again.top_ids.tolist() == out.top_ids.tolist() and again.rank.tolist() == out.rank.tolist()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = sg.logprobs(x, tokens, top=3, stream=side)
    side.synchronize()
    assert torch.equal(other.top_logprobs, out.top_logprobs) and torch.equal(other.entropy, out.entropy)
    plain = sg.logprobs(x)
    assert torch.isnan(plain.logprob).all() and (plain.rank == -1).all() and torch.equal(plain.entropy, out.entropy)


def test_sorted_rows_and_peaks_at_one_end(dev):
    # falling by id (as vocabularies ordered by frequency are), rising, and the likely ones side by side
    vocab = 60000
    x = torch.empty(3, vocab, device=dev)
    x[0] = torch.linspace(10, -10, vocab, device=dev)
    x[1] = x[0].flip(0)
    x[2] = -5.0 + 0.5 * torch.sin(torch.arange(vocab, device=dev).float())
    x[2, 30000:30100] = torch.linspace(6, 7, 100, device=dev)
    got = sg.logprobs(x, torch.tensor([100, 100, 30000], dtype=torch.int32, device=dev), top=64)
    lp = x.double().log_softmax(1)
    for r in range(3):
        order = torch.sort(x[r], descending=True, stable=True).indices
        assert torch.equal(got.top_ids[r].long(), order[:64])
        assert (got.top_logprobs[r].double() - lp[r, order[:64]]).abs().max() < (16 + 80 + 245 + 40) * U24
    assert got.rank.tolist() == [100, vocab - 101, 99]


def test_refusals(dev):
    x = torch.zeros(2, 100, device=dev)
    t = torch.zeros(2, dtype=torch.int32, device=dev)
    with pytest.raises(sg.SgError):
        sg.logprobs(x, t, top=65)
    with pytest.raises(sg.SgError):
        sg.logprobs(x[:, :10], t, top=11)
    with pytest.raises(TypeError):
        sg.logprobs(x, t.long())
    with pytest.raises(TypeError):
        sg.logprobs(x.double(), t)
    with pytest.raises(ValueError):
        sg.logprobs(x, t[:1])
    with pytest.raises(ValueError):
        sg.logprobs(x.t())
    with pytest.raises(ValueError):
        sg.logprobs(x, t, top=2, out=sg.LogProbs(2, 1, device=dev))
    assert sg.logprobs(x[:0], t[:0]).logprob.numel() == 0
