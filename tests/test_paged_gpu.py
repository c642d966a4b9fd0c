"""The paged decoder (spindle_b200.paged): the 4-bit cache operators together, as
a serving loop uses them."""
import numpy as np
import pytest
import torch

import decoder_util as D
import oracle as O
import spindle_b200 as sg
from spindle_b200.decoder import Decoder
from spindle_b200.paged import PagedDecoder

pytestmark = pytest.mark.gpu

DENSE = dict(dim=256, n_heads=4, n_kv_heads=2, head_dim=64, n_layers=2, vocab=512, max_seq=200, n_ff=512, rope_theta=1e4, rms_eps=1e-5,
             rope_neox=True)
MOE = dict(DENSE, n_heads=8, n_kv_heads=2, moe=dict(n_expert=8, n_used=2, n_ff=256), rope_neox=False, qk_norm=False)


def model(cfg, dev):
    dt = D.dtypes_for(cfg, embed=O.F16)
    w = {k: torch.from_numpy(np.ascontiguousarray(v)).to(dev) for k, v in D.host_weights(cfg, dt, seed=3).items()}
    return w, dt


def close(a, b):
    # the same tokens through other splits of the work: sums of another order, and now and then the code of an
    # activation that changes with them, 1 / 127 of its block's largest value
    return (a - b).abs().max() <= 0.02 * b.abs().max()


@pytest.mark.parametrize("cfg", [DENSE, MOE], ids=["dense", "moe"])
def test_requests_come_grow_and_end(dev, cfg):
    w, dt = model(cfg, dev)
    rng = np.random.default_rng(5)
    ts = {r: rng.integers(0, cfg["vocab"], 150).tolist() for r in range(4)}
    # each request alone, its tokens in one step
    alone = {}
    for r in ts:
        p = PagedDecoder(cfg, w, dt, dev, n_req=1, n_blocks=16, page=16)
        alone[r] = {k: p.step({0: ts[r][:k]} if not p.held[0] else {0: ts[r][p.held[0]:k]})["logits"][0] for k in (1, 40, 41, 150)}
    # together, in pieces, rows used again
    p = PagedDecoder(cfg, w, dt, dev, n_req=3, n_blocks=30, page=16)
    o = p.step({0: ts[0][:40], 2: ts[2][:1]}, top=5)
    assert o["requests"] == [0, 2] and close(o["logits"][0], alone[0][40]) and close(o["logits"][1], alone[2][1])
    lp = torch.log_softmax(o["logits"].double(), -1)
    assert torch.equal(o["probs"].top_ids[:, 0].long(), o["next"]) and (o["probs"].rank == 0).all()
    assert (o["probs"].logprob.double() - lp.amax(-1)).abs().max() < 1e-5
    o = p.step({0: ts[0][40:41], 1: ts[1][:40], 2: ts[2][1:40]})
    assert close(o["logits"][0], alone[0][41]) and close(o["logits"][1], alone[1][40]) and close(o["logits"][2], alone[2][40])
    o = p.step({2: ts[2][40:150]}, end=[0])
    assert close(o["logits"][0], alone[2][150])
    o = p.step({0: ts[3][:41], 1: ts[1][40:41]})                      # row 0 anew, on blocks given back
    assert close(o["logits"][0], alone[3][41]) and close(o["logits"][1], alone[1][41])
    with pytest.raises(ValueError):
        p.step({0: ts[3] + ts[2]})                                    # past max_seq
    with pytest.raises(RuntimeError):
        p.step({0: ts[3][41:150], 1: ts[1][:150]}, end=[])            # 30 blocks are not enough
    sg.device_status()


def test_near_the_f16_cache(dev):
    # the whole decoder with its f16 cache: K and V to 4 bits are off by about 8 % of their spread, attention
    # averages that, and the direction of the logits stays
    w, dt = model(DENSE, dev)
    toks = np.random.default_rng(8).integers(0, DENSE["vocab"], 120).tolist()
    full = Decoder(DENSE, w, dt, dev)
    want, _ = full.forward_batch(toks, 0, n_max=128)
    got = PagedDecoder(DENSE, w, dt, dev, n_req=1, n_blocks=8, page=32).step({0: toks})["logits"][0]
    assert torch.nn.functional.cosine_similarity(got.double(), want[-1].double(), dim=0) > 0.95


def test_example_runs(dev, capsys):
    from spindle_b200 import paged
    paged.main()
    assert "step 7 request 0" in capsys.readouterr().out
