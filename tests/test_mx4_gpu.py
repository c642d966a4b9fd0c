"""Microscaled 4-bit matrices on the GPU: rows quantized and read back, products."""
import pytest
import torch

import mx4_util as U
import spindle_b200 as sg

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def rand(dev, *shape, seed=0, spread=0.0):
    g = gen(dev, seed)
    x = torch.randn(*shape, device=dev, generator=g)
    return x * torch.exp(spread * torch.randn(*shape[:-1], 1, device=dev, generator=g)) if spread else x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (128, 256), (129, 288), (500, 4064)])
def test_quantize_and_back(dev, dtype, rows, cols):
    x = rand(dev, rows, cols, seed=rows, spread=2.0).to(dtype)
    m = sg.mx4_quantize(x)
    got = sg.mx4_dequantize(m)
    want = U.quantized(x)
    assert torch.equal(got.double(), want)
    for t in TYPES:
        assert torch.equal(sg.mx4_dequantize(m, dtype=t), want.to(t))
    # what is padding is zero
    n = -(-cols // 256)
    tiles = m.data.view(-1, n, 128 * 128 + 1024)
    codes = tiles[..., :128 * 128].unflatten(-1, (128, 8, 16))[-1, -1]
    r = torch.arange(128, device=dev)
    chunk = (torch.arange(8, device=dev) ^ (r[:, None] & 7))
    past = (chunk >= cols % 256 // 32) if cols % 256 else torch.zeros_like(chunk, dtype=torch.bool)
    past |= (r >= (rows % 128 or 128))[:, None]
    assert codes[past].count_nonzero() == 0


def test_quantize_strides_and_experts(dev):
    x = rand(dev, 3, 70, 2, 320, seed=1).half()
    for t in (x[:, :, 0], x[:, :, 1]):  # rows and experts any distance apart
        assert torch.equal(sg.mx4_dequantize(sg.mx4_quantize(t)).double(), U.quantized(t.contiguous()))
    y = rand(dev, 60, 331, seed=2)
    for off in (0, 1, 2, 3):            # rows without 16-byte alignment
        t = y[:, off:off + 320]
        m = sg.mx4_quantize(t)
        assert torch.equal(sg.mx4_dequantize(m).double(), U.quantized(t.contiguous()))
        out = torch.full((60, 340), 7.0, device=dev)
        sg.mx4_dequantize(m, out=out[:, off:off + 320])
        assert torch.equal(out[:, off:off + 320].double(), U.quantized(t.contiguous()))
        assert (out[:, :off] == 7).all() and (out[:, off + 320:] == 7).all()
    again = sg.Mx4(60, 320, device=dev)
    assert sg.mx4_quantize(y[:, :320], out=again) is again and torch.equal(again.data, sg.mx4_quantize(y[:, :320].contiguous()).data)


def test_quantize_edges(dev):
    big, tiny = 3.0e38, 2.0 ** -149
    x = torch.zeros(12, 64, device=dev)
    x[0, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])   # every tie
    x[1, :8] = -x[0, :8]
    x[2, 0], x[2, 1] = 7.0, 5.0
    x[3, 0], x[3, 1] = 6.9999995, 5.0
    x[4, 0] = tiny
    x[5, 0], x[5, 1] = 2.0 ** -126, tiny
    x[6, 0] = 2.5e38
    x[7, 5], x[7, 40] = float("nan"), 3.0
    x[8, 5], x[8, 40] = float("inf"), 3.0
    x[9, 5] = -float("inf")
    x[10, :] = -0.0
    x[11, :32] = torch.linspace(-6, 6, 32)
    got, want = sg.mx4_dequantize(sg.mx4_quantize(x)), U.quantized(x)
    assert torch.equal(torch.nan_to_num(got.double(), nan=99.0), torch.nan_to_num(want, nan=99.0))
    assert got[7, :32].isnan().all() and got[7, 40] == 3 and got[8, :32].isnan().all() and got[9, 33:].count_nonzero() == 0
    assert torch.isinf(sg.mx4_dequantize(sg.mx4_quantize(torch.full((1, 32), big, device=dev)))).all()  # 2^128, as the header says


SHAPES = [(1, 32, 1), (1, 256, 128), (1, 4096, 300), (2, 4096, 129), (3, 288, 77), (4, 14336, 513), (5, 96, 4096), (8, 2048, 768), (9, 4096, 1000),
          (16, 512, 128), (17, 1024, 2000), (32, 14336, 640), (33, 4096, 300), (64, 2080, 130), (100, 768, 2048), (128, 4096, 256), (129, 1056, 513),
          (255, 4096, 128), (257, 512, 1024), (1000, 2048, 1000), (2049, 1024, 300)]


@pytest.mark.parametrize("rows,cols,n", SHAPES)
def test_matmul(dev, rows, cols, n):
    x, w = rand(dev, rows, cols, seed=rows, spread=1.0), rand(dev, n, cols, seed=n, spread=0.5) * cols ** -0.5
    up = rand(dev, n, cols, seed=n + 1) * cols ** -0.5
    W, V = sg.mx4_quantize(w), sg.mx4_quantize(up)
    wq, vq = U.quantized(w), U.quantized(up)
    for dtype in TYPES:
        t = x.to(dtype)
        xq = U.quantized(t)
        want, bound = U.product(xq, wq)
        assert U.close(sg.mx4_matmul(t, W), want, bound)
        want, bound = U.product(xq, wq, vq)
        assert U.close(sg.mx4_matmul(t, W, up=V, dtype=torch.float32), want, bound)
    assert torch.equal(sg.mx4_matmul(x, W), sg.mx4_matmul(x, W))
    sg.device_status()


@pytest.mark.parametrize("rows", [1, 3, 20, 200, 600])
def test_matmul_strides(dev, rows):
    base = rand(dev, rows, 1100, seed=3)
    w = rand(dev, 300, 1024, seed=4) * 0.03
    W, wq = sg.mx4_quantize(w), U.quantized(w)
    for off in (0, 1, 8, 75):
        x = base[:, off:off + 1024]
        want, bound = U.product(U.quantized(x.contiguous()), wq)
        for dtype in TYPES:
            out = torch.full((rows + 2, 311), 7.0, dtype=dtype, device=dev)
            y = sg.mx4_matmul(x, W, out=out[1:-1, 5:305])
            assert U.close(y, want, bound)
            rest = out.clone()
            rest[1:-1, 5:305] = 7.0
            assert (rest == 7).all()  # nothing else is written
    sg.device_status()


@pytest.mark.parametrize("rows", [2, 200, 600])
@pytest.mark.parametrize("n", [1, 127, 258, 301])
def test_matmul_rows_of_results(dev, rows, n):
    # rows of results that begin on 16 bytes, on 4, on 2, and alternate
    x, w = rand(dev, rows, 320, seed=rows), rand(dev, n, 320, seed=n) * 0.05
    W = sg.mx4_quantize(w)
    want, bound = U.product(U.quantized(x), U.quantized(w))
    for dtype in TYPES:
        for off, ld in ((0, 320), (2, 320), (0, 314), (1, 320), (1, 313), (3, 314)):
            out = torch.full((rows + 1, ld), 7.0, dtype=dtype, device=dev)
            assert U.close(sg.mx4_matmul(x, W, out=out[:-1, off:off + n]), want, bound)
            out[:-1, off:off + n] = 7.0
            assert (out == 7).all()
    sg.device_status()


@pytest.mark.parametrize("rows", [1, 4, 16, 40, 300])
def test_matmul_nonfinite_rows_stay_apart(dev, rows):
    x, w = rand(dev, rows, 512, seed=5), rand(dev, 200, 512, seed=6)
    w[17, 300] = float("nan")
    bad = list(range(0, rows, 3))
    x[bad[::2], 100] = float("nan")
    x[bad[1::2], 300] = float("inf")
    y = sg.mx4_matmul(x, sg.mx4_quantize(w))
    nan = torch.zeros(rows, 200, dtype=torch.bool, device=dev)
    nan[bad] = True
    nan[:, 17] = True
    assert torch.equal(y.isnan(), nan)


@pytest.mark.parametrize("rows", [1, 30, 300])
def test_matmul_of_zeros_and_far_scales(dev, rows):
    w = rand(dev, 130, 256, seed=7)
    assert sg.mx4_matmul(torch.zeros(rows, 256, device=dev), sg.mx4_quantize(w)).count_nonzero() == 0
    # products of far scales are as in f32
    x = rand(dev, rows, 256, seed=8)
    want, bound = U.product(U.quantized(x * 2.0 ** 90), U.quantized(w * 2.0 ** -100))
    assert U.close(sg.mx4_matmul(x * 2.0 ** 90, sg.mx4_quantize(w * 2.0 ** -100)), want, bound)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_matmul_at_the_ends_of_the_scales(dev, rows):
    # scale bytes down to 0 (2^-127) and up to 252: products of the smallest and the largest, and of the smallest alone
    x, w = rand(dev, rows, 256, seed=8), rand(dev, 140, 256, seed=9) * 0.0625
    for a, b in ((-124, 120), (-123, 126), (120, -124), (-80, -60)):
        xs, ws = x * 2.0 ** a, w * 2.0 ** b
        want, bound = U.product(U.quantized(xs), U.quantized(ws))
        # (results below f32's normal numbers may be cut off)
        assert U.close(sg.mx4_matmul(xs, sg.mx4_quantize(ws)), want, bound + 2.0 ** -126)


def test_matmul_into_its_own_rows(dev):
    for rows in (1, 40, 300):
        x, W = rand(dev, rows, 256, seed=rows), sg.mx4_quantize(rand(dev, 256, 256, seed=1) * 0.06)
        want = sg.mx4_matmul(x, W)
        assert sg.mx4_matmul(x, W, out=x) is x and torch.equal(x, want)


def test_matmul_past_two_to_the_31(dev):
    # more than 2^31 results, and rows that begin past 2^32 bytes
    rows, n = 17001, 130000
    x, w = rand(dev, rows, 64, seed=1), rand(dev, n, 64, seed=2) * 0.125
    y = sg.mx4_matmul(x, sg.mx4_quantize(w), dtype=torch.float16)
    for r in ([0, 1, 5000], [8191, 8192, 16519, 16520], [16800, 16999, 17000]):
        for f in (slice(0, 300), slice(65000, 65300), slice(n - 300, n)):
            want, bound = U.product(U.quantized(x[r]), U.quantized(w[f]))
            assert U.close(y[r, f], want, bound)
    del y
    torch.cuda.empty_cache()


def test_dequantize_past_two_to_the_31(dev):
    rows, cols = 70001, 32768
    x = torch.zeros(rows, cols, dtype=torch.float16, device=dev)
    some = [0, 65535, 65536, 65537, 70000]
    x[some] = rand(dev, len(some), cols, seed=3).half()
    m = sg.mx4_quantize(x)
    want = U.quantized(x[some])
    y = sg.mx4_dequantize(m, out=x)
    assert torch.equal(y[some].double(), want) and y[1:65535:100].count_nonzero() == 0
    del x, y, m
    torch.cuda.empty_cache()


def test_matmul_empty_and_refusals(dev):
    W = sg.mx4_quantize(rand(dev, 64, 256))
    assert sg.mx4_matmul(torch.zeros(0, 256, device=dev), W).shape == (0, 64)
    x = rand(dev, 4, 256)
    with pytest.raises(ValueError):
        sg.mx4_matmul(x[:, :128], W)
    with pytest.raises(ValueError):
        sg.mx4_matmul(x.cpu(), W)
    with pytest.raises(ValueError):
        sg.mx4_matmul(x.T.contiguous().T, W)
    with pytest.raises(ValueError):
        sg.mx4_matmul(x, W, out=torch.empty(4, 63, device=dev))
    with pytest.raises(ValueError):
        sg.mx4_matmul(x, W, up=sg.mx4_quantize(rand(dev, 63, 256)))
    with pytest.raises(ValueError):
        sg.mx4_matmul(x, W, out=torch.empty(4, 64, device=dev), dtype=torch.float16)
    with pytest.raises(TypeError):
        sg.mx4_matmul(x.double(), W)
    with pytest.raises(sg.SgError):
        sg.mx4_matmul(torch.cat([x] * 20), W, scratch=torch.empty(0, dtype=torch.uint8, device=dev))
    with pytest.raises(sg.SgError):
        sg.mx4_matmul(x, sg.mx4_quantize(rand(dev, 2, 64, 256)))  # experts
    with pytest.raises(sg.SgError):
        sg.mx4_quantize(torch.zeros(4, 100, device=dev))


def test_captured_and_on_other_streams(dev):
    w = rand(dev, 700, 1024, seed=9) * 0.03
    W = sg.mx4_quantize(w)
    for rows in (1, 16, 200):
        x = rand(dev, rows, 1024, seed=10 + rows)
        scratch, out = sg.mx4_scratch(W, rows), torch.empty(rows, 700, device=dev)
        want = sg.mx4_matmul(x, W)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            sg.mx4_matmul(x, W, out=out, scratch=scratch)
        x.copy_(rand(dev, rows, 1024, seed=50 + rows))
        g.replay()
        assert torch.equal(out, sg.mx4_matmul(x, W))
        # two streams at once, scratch of their own
        side = [torch.cuda.Stream() for _ in range(2)]
        xs = [rand(dev, rows, 1024, seed=70 + i) for i in range(2)]
        torch.cuda.synchronize()
        got = [sg.mx4_matmul(xs[i % 2], W, stream=side[i % 2]) for i in range(8)]
        torch.cuda.synchronize()
        for i, y in enumerate(got):
            assert torch.equal(y, sg.mx4_matmul(xs[i % 2], W))
        assert want.isfinite().all()
    sg.device_status()
