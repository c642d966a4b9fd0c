"""The paged decoder on K-quants with a head of F16 rows: 4 bits where they are asked for."""
import numpy as np
import pytest
import torch

import spindle_b200 as sg
from spindle_b200.paged import Mx4Ffn, PagedDecoder
from test_paged_gpu import DENSE, MOE, model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cfg", [DENSE, MOE], ids=["dense", "moe"])
def test_a_head_of_rows(dev, cfg):
    w, dt = model(cfg, dev)
    head = (torch.randn(cfg["vocab"], cfg["dim"], device=dev, generator=torch.Generator(device=dev).manual_seed(1)) * 0.05).half()
    toks = np.random.default_rng(1).integers(0, cfg["vocab"], 50).tolist()
    rows, kinds = dict(w, head=head.view(torch.uint8)), dict(dt, head=sg.F16)
    with pytest.raises(ValueError):
        PagedDecoder(cfg, rows, kinds, dev, n_req=1, n_blocks=16)
    got = PagedDecoder(cfg, rows, kinds, dev, n_req=1, n_blocks=16, mx4=True).step({0: toks})["logits"]
    own = PagedDecoder(cfg, dict(w, head=sg.mx4_quantize(head)), {k: v for k, v in dt.items() if k != "head"}, dev, n_req=1, n_blocks=16)
    assert torch.equal(own.step({0: toks})["logits"], got)
    # K-quants alone, up's dtype left out
    names = {"l%d.%s" % (i, n) for i in range(cfg["n_layers"]) for n in ("up", "up_exps")}
    a, b = (PagedDecoder(cfg, w, d, dev, n_req=1, n_blocks=16).step({0: toks})["logits"] for d in (dt, {k: v for k, v in dt.items() if k not in names}))
    assert torch.equal(a, b)
    sg.device_status()


@pytest.mark.parametrize("n", [3, 300])
def test_the_router_is_whole_f32(dev, n):
    # torch's switch for TF32 products changes no token's experts, and is left as it was
    g = torch.Generator(device=dev).manual_seed(n)
    dim, ff, e = 512, 64, 64
    gate, up, down = (sg.mx4_quantize(torch.randn(e, a, b, device=dev, generator=g) * b ** -0.5) for a, b in ((ff, dim), (ff, dim), (dim, ff)))
    x, router = torch.randn(n, dim, device=dev, generator=g), torch.randn(e, dim, device=dev, generator=g)
    ffn = Mx4Ffn(gate, up, down, router=router, moe=dict(n_expert=e, n_used=8, n_ff=ff), n_max=n)
    want, weights = ffn(x), ffn.plan.weights.clone()
    m = torch.backends.cuda.matmul
    was = m.fp32_precision
    try:
        for on in ("tf32", "ieee"):
            m.fp32_precision = on
            assert torch.equal(ffn(x), want) and torch.equal(ffn.plan.weights, weights) and m.fp32_precision == on
    finally:
        m.fp32_precision = was
