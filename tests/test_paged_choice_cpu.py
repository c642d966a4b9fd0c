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
