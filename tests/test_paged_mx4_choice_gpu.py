"""The paged decoder on K-quants with a head of F16 rows: 4 bits where they are asked for."""
import numpy as np
import pytest
import torch

import spindle_b200 as sg
from spindle_b200.paged import PagedDecoder
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
