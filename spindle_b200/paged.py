"""Serving many requests from one 4-bit cache: a decoder whose requests come,
grow and end between steps, on the paged operators (kv4_plan, kv4_append,
kv4_attention, logprobs) and the framework's own projections (matmul_batch),
feed-forward layers (moe_forward_batch) and LM head.  The weights are named as
for decoder.Decoder; the embedding is F32 or F16 rows.  A matrix that is given as
an Mx4 is multiplied in microscaled 4 bits, weights and activations (mx4_matmul), all
tokens of a step in one call; a layer's experts too, sorted by expert (moe_route,
mx4_experts, moe_combine).  F32 and F16 rows become an Mx4 where the caller asks for it
(mx4=True); in a model without K-quants they do unless the caller forbids it
(mx4=False), with a warning.

    p = PagedDecoder(cfg, weights, dtypes, device, n_req=8, n_blocks=512)
    out = p.step({0: prompt_a, 3: prompt_b})        # tokens of the requests that go on
    out = p.step({0: [token], 3: [token]}, end=[5]) # and requests that end

`python -m spindle_b200.paged` runs it on a small random model."""
import warnings

import torch

from . import F16, F32, Moe, matmul_batch, moe_forward_batch, repack_tiled16
from .kv4 import LOGPROBS_TOP_MAX, Kv4Cache, Kv4Plan, LogProbs, kv4_append, kv4_attention, kv4_attention_scratch, kv4_plan, logprobs
from .mx4 import MoePlan, Mx4, moe_combine, moe_route, mx4_experts, mx4_matmul, mx4_quantize

BATCH = 128  # tokens of one batch GEMM or expert pass


def _router_logits(x, router):
    """x router^T in whole f32, as the K-quant layers' router has it, whatever torch's switches for faster f32 products say:
    a logit off by TF32's 2^-11 chooses other experts."""
    m = torch.backends.cuda.matmul
    was = m.fp32_precision
    if was in ("ieee", "none"):
        return x @ router.T
    m.fp32_precision = "ieee"
    try:
        return x @ router.T
    finally:
        m.fp32_precision = was


class Mx4Ffn:
    """A feed-forward layer in microscaled 4 bits: silu(x gate) * (x up), down; with a
    router a mixture of experts (moe: n_expert, n_used, norm, prune), n_max tokens at
    a time."""

    def __init__(self, gate, up, down, router=None, moe=None, n_max=0):
        self.gate, self.up, self.down, self.router, self.moe = gate, up, down, router, moe
        if (gate.experts, gate.rows, gate.cols) != (up.experts, up.rows, up.cols) or (down.experts, down.cols) != (gate.experts, gate.rows):
            raise ValueError("gate, up and down do not fit together")
        if moe:
            self.plan = MoePlan(n_max, moe["n_used"], moe["n_expert"], device=gate.data.device)

    def __call__(self, x):
        if not self.moe:
            return mx4_matmul(mx4_matmul(x, self.gate, up=self.up), self.down)
        p = moe_route(_router_logits(x, self.router), self.plan, norm=self.moe.get("norm", True), prune=self.moe.get("prune", 0.0))
        return moe_combine(mx4_experts(mx4_experts(x, self.gate, p, up=self.up), self.down, p), p)


class PagedDecoder:
    """n_req request rows over n_blocks blocks of `page` positions a layer; each
    request at most max_seq positions (cfg).  mx4: whether matrices of F32 or F16 rows
    become Mx4 ones (about 16 % rms off a product); None: where no matrix is a K-quant.
    dtypes needs no entry for an Mx4, nor for `up` (gate's then)."""

    def __init__(self, cfg, weights, dtypes, device, n_req, n_blocks, page=64, max_tokens=4096, mx4=None):
        c = self.cfg = dict(cfg)
        self.dev, self.n_req, self.n_blocks, self.page, self.max_tokens = device, n_req, n_blocks, page, max_tokens
        dim, hd = c["dim"], c["head_dim"]
        self.hq, self.hk, self.hd = c["n_heads"], c["n_kv_heads"], hd
        self.w = weights
        if dtypes["embed"] not in (F32, F16):
            raise ValueError("the embedding must be F32 or F16 rows")
        self.embed = weights["embed"].view(torch.float32 if dtypes["embed"] == F32 else torch.float16).view(c["vocab"], dim)

        def dtype(name):
            return None if isinstance(weights[name], Mx4) else dtypes[name if name in dtypes or ".up" not in name else name.replace(".up", ".gate")]
        ffn_names = ["gate_exps", "up_exps", "down_exps"] if c.get("moe") else ["gate", "up", "down"]
        kinds = {n: dtype(n) for n in ["head"] + ["l%d.%s" % (i, n) for i in range(c["n_layers"]) for n in ["wq", "wk", "wv", "wo"] + ffn_names]}
        rows = [n for n, k in kinds.items() if k in (F32, F16)]
        if rows and not mx4:
            if mx4 is False or any(k not in (None, F32, F16) for k in kinds.values()):
                raise ValueError("%s: F32 or F16 rows, which are served in microscaled 4 bits; that is asked for by mx4=True" % rows[0])
            warnings.warn("F32 and F16 matrices are served in microscaled 4 bits, weights and activations (mx4=True asks for it, mx4=False forbids it)",
                          stacklevel=2)

        def in4(name, *shape):
            """The matrix (or a layer's experts) if it is one in microscaled 4 bits, else None."""
            w = weights[name]
            if isinstance(w, Mx4):
                if (w.experts, w.rows, w.cols) != ((1,) + shape)[-3:]:
                    raise ValueError("%s must be a matrix %s" % (name, shape))
                return w
            if kinds[name] not in (F32, F16):
                return None
            return mx4_quantize(w.view(torch.float32 if kinds[name] == F32 else torch.float16).view(*shape))

        def mat(name, rows, cols):
            return in4(name, rows, cols) or repack_tiled16(dtypes[name], weights[name], rows, cols)

        self.layers = []
        for i in range(c["n_layers"]):
            p, moe = "l%d." % i, c.get("moe")
            ff, each = (moe["n_ff"], (moe["n_expert"],)) if moe else (c["n_ff"], ())
            mats = [in4(p + n, *each, *s) for n, s in zip(ffn_names, ((ff, dim), (ff, dim), (dim, ff)))]
            if any(m is not None for m in mats):
                if any(m is None for m in mats):
                    raise ValueError("gate, up and down of a layer are all in microscaled 4 bits or none of them")
                ffn = Mx4Ffn(*mats, router=weights[p + "router"].float().view(moe["n_expert"], dim) if moe else None, moe=moe, n_max=max_tokens)
            elif moe:
                ffn = Moe.pack(weights[p + "router"].float(), weights[p + "gate_exps"], weights[p + "up_exps"],
                               weights[p + "down_exps"], dtypes[p + "gate_exps"], dtypes[p + "down_exps"], moe["n_expert"],
                               moe["n_used"], dim, moe["n_ff"], norm=moe.get("norm", True), moe_prune=moe.get("prune", 0.0))
            else:  # a dense layer is a mixture of one expert
                ffn = Moe.pack(torch.zeros(1, dim, device=device), weights[p + "gate"], weights[p + "up"], weights[p + "down"],
                               dtypes[p + "gate"], dtypes[p + "down"], 1, 1, dim, c["n_ff"])
            self.layers.append(dict(
                wq=mat(p + "wq", self.hq * hd, dim), wk=mat(p + "wk", self.hk * hd, dim), wv=mat(p + "wv", self.hk * hd, dim),
                wo=mat(p + "wo", dim, self.hq * hd), ffn=ffn, cache=Kv4Cache(n_blocks, self.hk, hd, page, device=device)))
        self.head = mat("head", c["vocab"], dim)
        self.plan = Kv4Plan(n_req, max_tokens, page, n_blocks, device=device)
        self.tables = torch.full((n_req, -(-c["max_seq"] // page)), -1, dtype=torch.int32, device=device)
        self.ctx = torch.zeros(n_req, dtype=torch.int32, device=device)
        self.held = [0] * n_req  # the same on the host, to refuse what does not fit
        self.scratch = kv4_attention_scratch(device)
        half = torch.arange(hd // 2, device=device, dtype=torch.float64)
        self.freq = (c["rope_theta"] ** (-2.0 * half / hd)).float()

    def _norm(self, x, w):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + self.cfg["rms_eps"]) * w

    def _mm(self, m, x):
        if isinstance(m, Mx4):
            return mx4_matmul(x, m)
        t, mat = m
        out = torch.empty(x.shape[0], mat.rows, dtype=torch.float32, device=x.device)
        for a in range(0, x.shape[0], BATCH):
            matmul_batch(t, mat, x[a:a + BATCH], out=out[a:a + BATCH])
        return out

    def _rope(self, x, cos, sin):
        if self.cfg.get("rope_neox", True):
            a, b = x.chunk(2, -1)
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)

    def step(self, tokens, end=(), top=0):
        """One step: tokens maps a request row to its new tokens (a prompt or a part
        of one, or the token that follows); the requests in `end` give their blocks
        back (their rows start anew with the next tokens).  Returns a dict: for the
        requests with tokens, in rising order, `requests` (list), `logits` [n, vocab]
        after their last token, `next` (greedy, int64) and `probs`, the LogProbs of
        the greedy tokens with `top` alternatives."""
        new, end, vocab = [0] * self.n_req, set(end), self.cfg["vocab"]
        # (all of it before the plan, which changes what the requests hold)
        if not 0 <= top <= min(LOGPROBS_TOP_MAX, vocab):
            raise ValueError("top must be 0 to %d" % min(LOGPROBS_TOP_MAX, vocab))
        if any(not 0 <= r < self.n_req for r in end | set(tokens)):
            raise ValueError("requests are numbered 0 to %d" % (self.n_req - 1))
        tokens = {r: [int(t) for t in ts] for r, ts in tokens.items()}
        for r, ts in tokens.items():
            if any(not 0 <= t < vocab for t in ts):
                raise ValueError("request %d has a token outside the vocabulary" % r)
            if r in end:
                raise ValueError("request %d cannot end and go on in one step" % r)
            if self.held[r] + len(ts) > self.cfg["max_seq"]:
                raise ValueError("request %d would pass max_seq" % r)
            new[r] = len(ts)
        if sum(new) > self.max_tokens:
            raise ValueError("more than max_tokens new tokens")
        blocks = lambda n: -(-n // self.page)  # noqa: E731
        if sum(blocks(h + a) for h, a in zip(self.held, new)) > self.n_blocks:  # (what ends now is free from the next step on)
            raise RuntimeError("the cache has no free blocks for this step")
        for r in end:
            new[r] = -1
        p = kv4_plan(self.plan, self.ctx, torch.tensor(new, dtype=torch.int32, device=self.dev), self.tables)
        self.ctx = p.seq.clone()
        for r in range(self.n_req):
            self.held[r] = 0 if new[r] < 0 else self.held[r] + new[r]
        go = sorted(r for r in tokens if new[r] > 0)
        n = sum(new[r] for r in go)
        if n == 0:
            return None
        ids = torch.tensor([t for r in go for t in tokens[r]], dtype=torch.long, device=self.dev)
        c, slots = self.cfg, p.slots[:n]
        angle = p.pos[:n, None].float() * self.freq
        cos, sin = angle.cos()[:, None], angle.sin()[:, None]
        x = self.embed[ids].float() * c.get("embedding_scale", 1.0)
        scale = c.get("attn_scale", 0.0) or self.hd ** -0.5
        most = max(new)
        for i, y in enumerate(self.layers):
            w = lambda name: self.w.get("l%d.%s" % (i, name))  # noqa: E731,B023
            h = self._norm(x, w("attn_norm"))
            q, k, v = (self._mm(y[m], h).view(n, -1, self.hd) for m in ("wq", "wk", "wv"))
            if w("q_norm") is not None:
                q, k = self._norm(q, w("q_norm")), self._norm(k, w("k_norm"))
            q, k = self._rope(q, cos, sin), self._rope(k, cos, sin)
            kv4_append(y["cache"], k, v, slots)
            o = kv4_attention(y["cache"], q.contiguous(), p.cu, p.seq, self.tables, scale=scale, max_new=most, scratch=self.scratch)
            x = x + self._mm(y["wo"], o.view(n, -1)) * c.get("residual_scale", 1.0)
            h = self._norm(x, w("ffn_norm")).contiguous()
            if isinstance(y["ffn"], Mx4Ffn):
                f = y["ffn"](h)
            else:
                f = torch.empty_like(x)
                for a in range(0, n, BATCH):
                    moe_forward_batch(y["ffn"], h[a:a + BATCH], out=f[a:a + BATCH])
            x = x + f * c.get("residual_scale", 1.0)
        last = torch.tensor([sum(new[q] for q in go if q <= r) - 1 for r in go], device=self.dev)
        logits = self._mm(self.head, self._norm(x[last], self.w["out_norm"]).contiguous())
        nxt = logits.argmax(-1)
        return {"requests": go, "logits": logits, "next": nxt, "probs": logprobs(logits, nxt.int(), top=top, out=LogProbs(len(go), top, self.dev))}


def serve(d):
    """A few requests served together, printed."""
    out = d.step({0: list(range(5, 45)), 2: [7, 8, 9]}, top=3)
    for step in range(8):
        ids = out["next"].tolist()
        for r, t, lp, ent in zip(out["requests"], ids, out["probs"].logprob.tolist(), out["probs"].entropy.tolist()):
            print("step %d request %d token %4d logprob %.3f entropy %.3f" % (step, r, t, lp, ent))
        nxt = {r: [t] for r, t in zip(out["requests"], ids)}
        if step == 3:
            nxt[1] = [11, 12, 13, 14]  # another request joins
        if step == 5:
            del nxt[2]                 # and one ends
        out = d.step(nxt, end=[2] if step == 5 else [], top=3)


def main():
    """Two small random models: K-quants, and a mixture of experts in microscaled 4 bits."""
    from . import Q4_K, Q6_K, quantize_weights
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(0)
    dense = dict(dim=512, n_heads=8, n_kv_heads=2, head_dim=64, n_layers=2, vocab=1024, max_seq=512, n_ff=768, rope_theta=1e6,
                 rms_eps=1e-6, rope_neox=True)
    for cfg in (dense, dict(dense, moe=dict(n_expert=16, n_used=4, n_ff=256))):
        dim, w, dt = cfg["dim"], {}, {}

        def mat(name, kind, *shape):
            x = torch.randn(*shape, device=dev, generator=g) * 0.05
            w[name], dt[name] = (mx4_quantize(x), None) if cfg.get("moe") else (quantize_weights(kind, x), kind)  # noqa: B023

        w["embed"], dt["embed"] = torch.randn(cfg["vocab"], dim, device=dev, generator=g).half().view(torch.uint8), F16
        mat("head", Q6_K, cfg["vocab"], dim)
        w["out_norm"] = torch.ones(dim, device=dev)
        for i in range(cfg["n_layers"]):
            p, moe = "l%d." % i, cfg.get("moe")
            w[p + "attn_norm"], w[p + "ffn_norm"] = torch.ones(dim, device=dev), torch.ones(dim, device=dev)
            for name, rows, cols in (("wq", 512, dim), ("wk", 128, dim), ("wv", 128, dim), ("wo", dim, 512)):
                mat(p + name, Q4_K, rows, cols)
            ff, each, s = (moe["n_ff"], (moe["n_expert"],), "_exps") if moe else (cfg["n_ff"], (), "")
            for name, rows, cols in (("gate", ff, dim), ("up", ff, dim), ("down", dim, ff)):
                mat(p + name + s, Q4_K, *each, rows, cols)
            if moe:
                w[p + "router"] = torch.randn(moe["n_expert"], dim, device=dev, generator=g) * 0.05
        print("experts in microscaled 4 bits:" if cfg.get("moe") else "K-quants:")
        serve(PagedDecoder(cfg, w, dt, dev, n_req=4, n_blocks=64, page=16))


if __name__ == "__main__":
    main()
