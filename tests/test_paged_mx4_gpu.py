"""The paged decoder on matrices in microscaled 4 bits: projections, feed-forward layers
and experts together, as a serving loop uses them."""
import numpy as np
import pytest
import torch

import mx4_util as U
import spindle_b200 as sg
from spindle_b200.paged import Mx4Ffn, PagedDecoder

pytestmark = pytest.mark.gpu

DENSE = dict(dim=256, n_heads=4, n_kv_heads=2, head_dim=64, n_layers=2, vocab=512, max_seq=200, n_ff=512, rope_theta=1e4, rms_eps=1e-5,
             rope_neox=True)
MOE = dict(DENSE, n_heads=8, moe=dict(n_expert=8, n_used=2, n_ff=224), rope_neox=False)


def model(cfg, dev, as_rows=None):
    """Random weights: F16 (or F32) rows, or Mx4."""
    g = torch.Generator(device=dev).manual_seed(2)
    w, dt, dim, moe = {}, {}, cfg["dim"], cfg.get("moe")

    def mat(name, *shape):
        x = (torch.randn(*shape, device=dev, generator=g) * shape[-1] ** -0.5).half().to(as_rows or torch.float16)
        w[name], dt[name] = (x.view(torch.uint8), sg.F16 if as_rows == torch.float16 else sg.F32) if as_rows else (sg.mx4_quantize(x), None)
    w["embed"], dt["embed"] = torch.randn(cfg["vocab"], dim, device=dev, generator=g).half().view(torch.uint8), sg.F16
    mat("head", cfg["vocab"], dim)
    w["out_norm"] = 1 + 0.1 * torch.randn(dim, device=dev, generator=g)
    for i in range(cfg["n_layers"]):
        p, hd = "l%d." % i, cfg["head_dim"]
        w[p + "attn_norm"], w[p + "ffn_norm"] = (1 + 0.1 * torch.randn(dim, device=dev, generator=g) for _ in range(2))
        for name, heads in (("wq", cfg["n_heads"]), ("wk", cfg["n_kv_heads"]), ("wv", cfg["n_kv_heads"])):
            mat(p + name, heads * hd, dim)
        mat(p + "wo", dim, cfg["n_heads"] * hd)
        each, ff, s = ((moe["n_expert"],), moe["n_ff"], "_exps") if moe else ((), cfg["n_ff"], "")
        for name, rows, cols in (("gate", ff, dim), ("up", ff, dim), ("down", dim, ff)):
            mat(p + name + s, *each, rows, cols)
        if moe:
            w[p + "router"] = torch.randn(moe["n_expert"], dim, device=dev, generator=g) * dim ** -0.5
    return w, dt


def decoder(cfg, dev, as_rows=None, **kw):
    return PagedDecoder(cfg, *model(cfg, dev, as_rows), dev, **dict(dict(n_req=3, n_blocks=40, page=16), **kw))


@pytest.mark.parametrize("cfg", [DENSE, MOE], ids=["dense", "moe"])
def test_rows_become_the_same_matrices(dev, cfg):
    toks = np.random.default_rng(1).integers(0, cfg["vocab"], 60).tolist()
    want = decoder(cfg, dev).step({1: toks})["logits"]
    for rows in (torch.float16, torch.float32):
        assert torch.equal(decoder(cfg, dev, rows).step({1: toks})["logits"], want)
    sg.device_status()


@pytest.mark.parametrize("cfg", [DENSE, MOE], ids=["dense", "moe"])
def test_together_and_in_pieces(dev, cfg):
    # the same tokens in other batches: the products are the same up to the order of their sums, but a sum's last bit can
    # move an activation to the next code, a sixth to a half of its size; that is rare, and the logits' direction stays
    rng = np.random.default_rng(5)
    ts = {r: rng.integers(0, cfg["vocab"], 120).tolist() for r in range(3)}
    alone = {r: decoder(cfg, dev, n_req=1, n_blocks=16).step({0: ts[r]})["logits"][0] for r in ts}
    p = decoder(cfg, dev)
    p.step({0: ts[0][:50], 2: ts[2][:119]})
    o = p.step({0: ts[0][50:], 1: ts[1], 2: ts[2][119:]}, top=4)
    assert o["requests"] == [0, 1, 2]
    for r in ts:
        assert torch.nn.functional.cosine_similarity(o["logits"][r].double(), alone[r].double(), dim=0) > 0.99
    assert torch.equal(o["probs"].top_ids[:, 0].long(), o["next"])
    sg.device_status()


@pytest.mark.parametrize("n", [1, 30, 500])
@pytest.mark.parametrize("prune", [0.0, 0.4])
def test_feed_forward_layers(dev, n, prune):
    g = torch.Generator(device=dev).manual_seed(n)
    dim, ff, e, k = 256, 160, 12, 4
    x = torch.randn(n, dim, device=dev, generator=g)
    gate, up, down = (torch.randn(e, a, b, device=dev, generator=g) * b ** -0.5 for a, b in ((ff, dim), (ff, dim), (dim, ff)))
    router = torch.randn(e, dim, device=dev, generator=g) * dim ** -0.5
    moe = dict(n_expert=e, n_used=k, n_ff=ff, prune=prune)
    got = Mx4Ffn(*(sg.mx4_quantize(t) for t in (gate, up, down)), router=router, moe=moe, n_max=n)(x)
    dense = Mx4Ffn(*(sg.mx4_quantize(t[0]) for t in (gate, up, down)))(x)
    xq, (gq, uq, dq) = U.quantized(x), (U.quantized(t) for t in (gate, up, down))

    def layer(rows, j):  # in 64 bits; the hidden values go to 4 bits as f32
        h = rows @ gq[j].T
        h = h * torch.sigmoid(h) * (rows @ uq[j].T)
        return U.quantized(h.float()) @ dq[j].T
    ids, weights = U.choice(x @ router.T, k, True, prune)
    want = torch.zeros(n, dim, dtype=torch.float64, device=dev)
    for t in range(n):
        for j, w in zip(ids[t].tolist(), weights[t].tolist()):
            if j >= 0:
                want[t] += w * layer(xq[t:t + 1], j)[0]
    for a, b in ((got, want), (dense, layer(xq, 0))):
        # (a hidden value at the edge of two codes may take the other one: few, one step of one of ff of them)
        assert (a.double() - b).norm() <= 1e-2 * b.norm()
        assert ((a.double() - b).abs() <= 1e-5 * b.abs().amax()).double().mean() > 0.9


def test_refusals(dev):
    w, dt = model(DENSE, dev)
    with pytest.raises(ValueError):
        PagedDecoder(dict(DENSE, n_ff=480), w, dt, dev, n_req=1, n_blocks=8)       # another shape than the matrices have
    q, qt = dict(w), dict(dt)
    q["l0.up"], qt["l0.up"] = sg.quantize_weights(sg.Q4_K, torch.randn(512, 256, device=dev)), sg.Q4_K
    with pytest.raises(ValueError):
        PagedDecoder(DENSE, q, qt, dev, n_req=1, n_blocks=8)                       # one of gate, up and down in another format
    for name, rows, cols in (("gate", 512, 256), ("up", 512, 256), ("down", 256, 512)):
        for i in range(2):
            q["l%d.%s" % (i, name)], qt["l%d.%s" % (i, name)] = sg.quantize_weights(sg.Q4_K, torch.randn(rows, cols, device=dev) * 0.05), sg.Q4_K
    assert PagedDecoder(DENSE, q, qt, dev, n_req=1, n_blocks=8).step({0: [1, 2, 3]})["logits"].isfinite().all()  # a mixed model
    with pytest.raises(ValueError):
        Mx4Ffn(w["l0.gate"], w["l0.up"], w["l0.gate"])
