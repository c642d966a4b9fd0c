"""CPU checks of how PagedDecoder takes the matrices that it is given, up to the first that goes
to the GPU."""
import pytest
import torch

from spindle_b200 import F16, F32, Q4_K, Q6_K, paged

CFG = dict(dim=256, n_heads=4, n_kv_heads=2, head_dim=64, n_layers=2, vocab=512, max_seq=200, n_ff=512, rope_theta=1e4, rms_eps=1e-5)
MOE = dict(CFG, moe=dict(n_expert=8, n_used=2, n_ff=256))


class Reached(Exception):
    """All matrices have been looked at: the first cache is made."""


class FakeMx4:
    def __init__(self, *shape):
        self.experts, self.rows, self.cols = ((1,) + shape)[-3:]


@pytest.fixture
def made(monkeypatch):
    """The matrices that are made of what is given, in order, without a GPU."""
    got = []

    def stop(*a, **kw):
        raise Reached

    def quantize(x):
        got.append(("mx4", x.dtype))
        return FakeMx4(*x.shape)
    monkeypatch.setattr(paged, "repack_tiled16", lambda kind, w, rows, cols: got.append(("repack", kind)))
    monkeypatch.setattr(paged, "Moe", type("Moe", (), dict(pack=lambda *a, **kw: got.append(("pack", a[4], a[5])))))
    monkeypatch.setattr(paged, "Mx4Ffn", lambda *a, **kw: got.append(("ffn4",)))
    monkeypatch.setattr(paged, "mx4_quantize", quantize)
    monkeypatch.setattr(paged, "Mx4", FakeMx4)
    monkeypatch.setattr(paged, "Kv4Cache", stop)
    return got


def shapes(cfg):
    dim, ff, each, s = cfg["dim"], cfg["n_ff"], (), ""
    if "moe" in cfg:
        ff, each, s = cfg["moe"]["n_ff"], (cfg["moe"]["n_expert"],), "_exps"
    out = dict(head=(cfg["vocab"], dim))
    for i in range(cfg["n_layers"]):
        p, q, k = "l%d." % i, cfg["n_heads"] * cfg["head_dim"], cfg["n_kv_heads"] * cfg["head_dim"]
        out.update({p + "wq": (q, dim), p + "wk": (k, dim), p + "wv": (k, dim), p + "wo": (dim, q), p + "gate" + s: each + (ff, dim),
                    p + "up" + s: each + (ff, dim), p + "down" + s: each + (dim, ff)})
    return out


def model(cfg, kind):
    """Weights of which kind(name) says what they are: a dtype, or "mx4"."""
    w, dt = dict(embed=torch.zeros(cfg["vocab"] * cfg["dim"], dtype=torch.float16).view(torch.uint8)), dict(embed=F16)
    for n, s in shapes(cfg).items():
        k, size = kind(n), torch.Size(s).numel()
        if k == "mx4":
            w[n] = FakeMx4(*s)
        else:
            w[n], dt[n] = torch.zeros(size * {F32: 4, F16: 2}.get(k, 0) or 16, dtype=torch.uint8), k
    for i in range(cfg["n_layers"]):
        w["l%d.router" % i] = torch.zeros(8, cfg["dim"])
    return w, dt


def make(cfg, w, dt, **kw):
    with pytest.raises(Reached):
        paged.PagedDecoder(cfg, w, dt, torch.device("cpu"), n_req=1, n_blocks=8, **kw)


@pytest.mark.parametrize("cfg", [CFG, MOE], ids=["dense", "moe"])
def test_up_needs_no_dtype(made, cfg):
    # the K-quant path takes gate's for both
    w, dt = model(cfg, lambda n: Q6_K if "down" in n else Q4_K)
    make(cfg, w, {n: k for n, k in dt.items() if ".up" not in n})
    assert made[0] == ("pack", Q4_K, Q6_K)


@pytest.mark.parametrize("kind", [F16, F32])
@pytest.mark.parametrize("name", ["head", "l0.wq", "l1.wo", "ffn"])
@pytest.mark.parametrize("cfg", [CFG, MOE], ids=["dense", "moe"])
def test_rows_in_a_model_of_k_quants(made, cfg, name, kind):
    # one matrix of F16 or F32 rows (or a layer's three): 4 bits are asked for, or it is refused before anything is made
    names = [n for n in shapes(cfg) if n.startswith(("l1.gate", "l1.up", "l1.down"))] if name == "ffn" else [name]
    w, dt = model(cfg, lambda n: kind if n in names else Q4_K)
    for kw in ({}, dict(mx4=None), dict(mx4=False)):
        with pytest.raises(ValueError, match="mx4=True"):
            paged.PagedDecoder(cfg, w, dt, torch.device("cpu"), n_req=1, n_blocks=8, **kw)
        assert made == []
    # beside matrices that the caller made into 4 bits as well
    w2, dt2 = model(cfg, lambda n: kind if n in names else "mx4" if n.startswith("l0") else Q4_K)
    with pytest.raises(ValueError, match="mx4=True"):
        paged.PagedDecoder(cfg, w2, dt2, torch.device("cpu"), n_req=1, n_blocks=8)
    assert made == []
    make(cfg, w, dt, mx4=True)


@pytest.mark.parametrize("cfg", [CFG, MOE], ids=["dense", "moe"])
def test_a_model_of_rows(made, cfg):
    w, dt = model(cfg, lambda n: F16)
    with pytest.warns(UserWarning, match="4 bits"):
        make(cfg, w, dt)
    n = len(made)
    assert ("mx4", torch.float16) in made and ("ffn4",) in made
    with pytest.raises(ValueError, match="mx4=True"):
        paged.PagedDecoder(cfg, w, dt, torch.device("cpu"), n_req=1, n_blocks=8, mx4=False)
    assert len(made) == n


@pytest.mark.parametrize("kw", [{}, dict(mx4=False), dict(mx4=True)])
@pytest.mark.parametrize("cfg", [CFG, MOE], ids=["dense", "moe"])
def test_what_the_caller_made_stays(made, cfg, kw, recwarn):
    # Mx4s, with K-quants beside them or without, need no entry in dtypes
    for kind in (lambda n: "mx4", lambda n: "mx4" if n.startswith(("l0.gate", "l0.up", "l0.down")) else Q4_K):
        make(cfg, *model(cfg, kind), **kw)
        assert made[0] == ("ffn4",) and not any(m[0] == "mx4" for m in made)
    w, dt = model(cfg, lambda n: Q4_K)
    make(cfg, w, dt, **kw)
    assert not recwarn.list


def test_up_of_another_kind(made):
    w, dt = model(CFG, lambda n: F16 if n == "l0.up" else Q4_K)
    with pytest.raises(ValueError):
        paged.PagedDecoder(CFG, w, dt, torch.device("cpu"), n_req=1, n_blocks=8, mx4=True)
