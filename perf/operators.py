"""The transformer operators of a training step around the optimizer, as timed and compared cases.

A model that trains with the low-bit optimizer takes its tokens in through an embedding table, mixes
them in attention layers, carries a residual stream through norms before and after each block, and
learns from labels or from a teacher's top logits.  A case names one of these operators (``op``), its
sizes, the type of its tensors (``dtype``) and how far it goes (``dir``):

``emb``    ``embedding_forward``, and ``embedding_backward`` into a dense gradient of the table
``norm``   ``norm_residual_forward`` / ``norm_residual_backward``: r = a x + gate * norm_post(block),
           h = norm_pre(r), with RMS or layer norms
``attn``   ``attention_forward`` / ``attention_backward``: causal softmax attention that sees a window of
           the last keys and a few first ones, with shared key heads and a mask of keys
``dist``   ``distill_loss_*``: T^2 KL(teacher's top-K || student) mixed with the labels' cross-entropy,
           and its gradient over the whole vocabulary

``dir``: ``fwd`` returns what the forward pass computes, ``train`` the forward pass and then the gradients
of its inputs, ``fused`` (dist) both from one call.
"""
import math
import os
import sys

import torch

own = False          # True: the framework's operators; False: their plain form

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stream-mm2026_amd")
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
NEG = float("-inf")


def listed():
    return [
        # A few tokens looked up in a full table, fp32 master weights into bf16 activations: the smallest call, launch latency.
        dict(name="emb_few", op="emb", dir="fwd", n=9, vocab=50257, d=768, dtype="f32", out="bf16", zipf=False, pad=False),
        # GPT-2 small's token table on one micro-batch of 8 x 1024: the table's dense fp32 gradient is what has to be written.
        dict(name="emb_gpt2", op="emb", dir="train", n=8192, vocab=50257, d=768, dtype="f32", out="f32", zipf=False, pad=False),
        # A 32000 x 4096 bf16 table under text-like (Zipf) tokens: a few rows gather thousands of gradients each.
        dict(name="emb_zipf", op="emb", dir="train", n=16384, vocab=32000, d=4096, dtype="bf16", out="bf16", zipf=True, pad=True),
        # Five positions of width 768 in fp32 with biases: a norm during evaluation, launch latency.
        dict(name="norm_few", op="norm", dir="fwd", n=5, d=768, dtype="f32", kind="layer", post=False, gate=0),
        # GPT-2 small's layer norm behind a residual sum, forward and backward: short rows.
        dict(name="norm_gpt2", op="norm", dir="train", n=8192, d=768, dtype="bf16", kind="layer", post=False, gate=0),
        # Width 4096, RMS norms before and after the block, a gate per channel: wide rows, the largest.
        dict(name="norm_4096", op="norm", dir="train", n=16384, d=4096, dtype="bf16", kind="rms", post=True, gate=1),
        # One new position over a long context: few rows, the key axis is all there is to split.
        dict(name="attn_one", op="attn", dir="fwd", b=2, hk=4, group=3, d=64, t=1, s=4097, window=0, sinks=0, pad=0, dtype="bf16"),
        # GPT-2 small's attention on one micro-batch, forward and backward.
        dict(name="attn_gpt2", op="attn", dir="train", b=8, hk=12, group=1, d=64, t=1024, s=1024, window=0, sinks=0, pad=0, dtype="bf16"),
        # Heads of 128, four to a key head, 8192 positions of which each sees the last 2048 and the first 4: long training rows, the largest.
        dict(name="attn_window", op="attn", dir="train", b=1, hk=8, group=4, d=128, t=8192, s=8192, window=2048, sinks=4, pad=0,
             dtype="bf16"),
        # Left-padded sequences of odd length with heads of 80 in fp16: rows that see nothing, partial tiles.
        dict(name="attn_ragged", op="attn", dir="train", b=5, hk=3, group=2, d=80, t=777, s=777, window=300, sinks=3, pad=210, dtype="f16"),
        # A handful of positions over a 32000 vocabulary in fp32, few teacher entries.
        dict(name="dist_few", op="dist", dir="train", n=7, vocab=32000, k=8, dtype="f32", temp=1.0, alpha=1.0, labels=False, banned=0),
        # GPT-2 small's logits of one micro-batch against a teacher's top 64 and the labels, gradient included: the largest bytes.
        dict(name="dist_gpt2", op="dist", dir="fused", n=8192, vocab=50257, k=64, dtype="bf16", temp=2.0, alpha=0.7, labels=True, banned=41),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges; sizes that would cost more than the largest listed case of their kind are halved until they do not."""
    op = rng.choice(["emb", "norm", "attn", "attn", "dist"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "emb":
        c = dict(op=op, dir=rng.choice(["fwd", "train", "train"]), n=_log(rng, 1, 65536), vocab=rng.choice([50257, 32000, _log(rng, 200, 200000)]),
                 d=rng.choice([768, 4096, 8 * _log(rng, 4, 512), _log(rng, 33, 1500)]), dtype=dtype, out=rng.choice([dtype, dtype, "bf16"]),
                 zipf=rng.random() < 0.5, pad=rng.random() < 0.5)
        shrink = "n"
        if c["vocab"] * c["d"] > 32000 * 4096:
            c["vocab"] = 32000 * 4096 // c["d"]
    elif op == "norm":
        c = dict(op=op, dir=rng.choice(["fwd", "train", "train"]), n=_log(rng, 1, 32768),
                 d=rng.choice([768, 4096, 8 * _log(rng, 4, 1000), _log(rng, 33, 4000)]), dtype=dtype, kind=rng.choice(["rms", "layer"]),
                 post=rng.random() < 0.6, gate=rng.choice([0, 1, 2]))
        c["n"] += c["n"] % 2 if c["gate"] == 2 else 0    # gate 2: one row of gates for each half of the positions
        shrink = "n"
    elif op == "attn":
        t = _log(rng, 1, 6000)
        c = dict(op=op, dir=rng.choice(["fwd", "train", "train"]), b=rng.randint(1, 8), hk=rng.randint(1, 12), group=rng.choice([1, 1, 2, 4, 7]),
                 d=rng.choice([64, 128, 8 * rng.randint(2, 16)]), t=t, s=t + rng.choice([0, 0, _log(rng, 1, 3000)]),
                 window=rng.choice([0, _log(rng, 1, 3000)]), sinks=rng.choice([0, 0, rng.randint(1, 70)]), pad=0, dtype=rng.choice(["bf16", "f16"]))
        if rng.random() < 0.4:
            c["pad"] = rng.randint(1, c["s"])
        shrink = "b"
    else:
        c = dict(op=op, dir=rng.choice(["fwd", "train", "fused", "fused"]), n=_log(rng, 1, 16384), vocab=rng.choice([50257, 32000, _log(rng, 300, 150000)]),
                 k=_log(rng, 1, 200), dtype=dtype, temp=rng.choice([1.0, 2.0, 4.0]), alpha=rng.choice([1.0, 0.7, 0.3]), labels=rng.random() < 0.6,
                 banned=rng.choice([0, rng.randint(1, 50)]))
        shrink = "n"
    most = {"emb": 0.8e9, "norm": 1.3e9, "attn": 2.0e9, "dist": 1.6e9}[op]
    while work(c)["bytes"] > most or work(c)["flops"] > 1.4e12 or _plain_bytes(c) > 9e9:
        if c[shrink] == 1:
            shrink = "hk"
        c[shrink] = max(1, c[shrink] // 2)
        if op == "norm" and c["gate"] == 2:
            c["n"] += c["n"] % 2
    return c


def _plain_bytes(c):
    """The largest array of the plain form."""
    return 4.0 * c["b"] * c["hk"] * c["group"] * c["t"] * c["s"] if c["op"] == "attn" else 0.0


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)


def _randn(gen, *shape, std=1.0, dtype=torch.float32):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for o in range(0, flat.numel(), 1 << 26):
        k = min(1 << 26, flat.numel() - o)
        flat[o:o + k] = torch.randn(k, device="cuda", generator=gen).mul_(std)
    return out


def _tokens(c, gen):
    v = c["vocab"]
    if not c["zipf"]:
        return torch.randint(0, v, (c["n"],), device="cuda", generator=gen)
    # log-uniform ranks (frequencies falling as 1 / rank), scattered over the table
    rank = torch.rand(c["n"], device="cuda", generator=gen, dtype=torch.float64).mul_(math.log(v)).exp_().long().clamp_(1, v) - 1
    return (rank * 7919 + 13) % v


def _pads(c):
    """How many first keys of each sequence are padding: spread from none to ``pad``."""
    return [(i * c["pad"]) // max(1, c["b"] - 1) if c["b"] > 1 else c["pad"] for i in range(c["b"])]


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt = DTYPE[c["dtype"]]
    s = dict(c=c)
    if c["op"] == "emb":
        s["tokens"] = _tokens(c, g)
        s["weight"] = _randn(g, c["vocab"], c["d"], std=0.02, dtype=dt)
        s["scale"] = math.sqrt(c["d"]) if c["pad"] else 1.0
        s["padding"] = 13 % c["vocab"] if c["pad"] else None      # the most frequent token of a Zipf draw
        if c["dir"] == "train":
            s["grad"] = _randn(g, c["n"], c["d"], std=1e-2, dtype=DTYPE[c["out"]])
    elif c["op"] == "norm":
        n, d = c["n"], c["d"]
        s["x"] = _randn(g, n, d, std=2.0, dtype=dt) + _randn(g, d, std=0.5).to(dt)
        s["block"] = _randn(g, n, d, std=0.7, dtype=dt) + (0.3 if c["kind"] == "layer" else 0.0)
        layer = c["kind"] == "layer"
        near1 = lambda: (1.0 + _randn(g, d, std=0.1)).to(dt)  # noqa: E731
        s["pre_weight"], s["pre_bias"] = near1(), _randn(g, d, std=0.1).to(dt) if layer else None
        s["post_weight"] = near1() if c["post"] else None
        s["post_bias"] = _randn(g, d, std=0.1).to(dt) if layer and c["post"] else None
        s["gate"] = _randn(g, c["gate"], d, std=0.5, dtype=dt) if c["gate"] else None
        s["scale"] = 0.9 if c["post"] else 1.0
        if c["dir"] == "train":
            s["dr"], s["dh"] = _randn(g, n, d, std=1e-2, dtype=dt), _randn(g, n, d, std=1e-2, dtype=dt)
    elif c["op"] == "attn":
        b, hk, h, d, t, S = c["b"], c["hk"], c["hk"] * c["group"], c["d"], c["t"], c["s"]
        if t == S:
            # one projection's output [b, t, (h + 2 hk) d], split and transposed as a model does
            qkv = _randn(g, b, t, (h + 2 * hk) * d, dtype=dt)
            q, k, v = (x.view(b, t, -1, d).transpose(1, 2) for x in qkv.split([h * d, hk * d, hk * d], dim=-1))
        else:
            q = _randn(g, b, t, h, d, dtype=dt).transpose(1, 2)
            k, v = (_randn(g, b, hk, S, d, dtype=dt) for _ in range(2))
        s.update(q=q, k=k, v=v, scale=d ** -0.5)
        s["mask"] = None
        if c["pad"]:
            s["mask"] = torch.arange(S, device="cuda")[None, :] >= torch.tensor(_pads(c), device="cuda")[:, None]
        if c["dir"] == "train":
            s["do"] = _randn(g, b, t, h, d, std=1e-2, dtype=dt).transpose(1, 2)
    else:
        n, v, k = c["n"], c["vocab"], c["k"]
        s["logits"] = _randn(g, n, v, std=2.5, dtype=dt)
        if c["banned"]:
            s["logits"][:, v - c["banned"]:] = NEG              # columns that the student never answers with
        live = v - c["banned"]
        # k different tokens a row: an arithmetic progression modulo the live vocabulary, with a few absent entries
        first = torch.randint(0, live, (n, 1), device="cuda", generator=g)
        stride = live // k
        s["ids"] = (first + stride * torch.arange(k, device="cuda")) % live
        s["teacher"] = torch.sort(_randn(g, n, k, std=3.0), dim=1, descending=True)[0].to(dt)
        rows = torch.rand(n, device="cuda", generator=g)
        if k > 1:
            s["ids"][rows < 0.2, k - 1] = -1                    # nucleus-cut rows keep fewer entries
        s["labels"] = torch.randint(0, live, (n,), device="cuda", generator=g) if c["labels"] else None
        if c["labels"]:
            s["labels"][rows > 0.9] = -100                      # positions without a label
            s["ids"][rows > 0.95] = -1                          # padding: neither label nor teacher
        # the gradient of the mean loss; fp16 training scales its losses
        s["drow"] = torch.full((n,), (4096.0 if c["dtype"] == "f16" else 1.0) / n, device="cuda")
    return s


# ------------------------------------------------------------------ the plain forms, in 32 bits
def _plain_emb(s):
    c = s["c"]
    out = (s["weight"][s["tokens"]].float() * s["scale"]).to(DTYPE[c["out"]])
    if c["dir"] == "fwd":
        return {"out": out}
    g = s["grad"].float() * s["scale"]
    if s["padding"] is not None:
        g = torch.where((s["tokens"] == s["padding"])[:, None], torch.zeros((), device="cuda"), g)
    dw = torch.zeros(c["vocab"], c["d"], device="cuda").index_add_(0, s["tokens"], g)
    return {"out": out, "dweight": dw.to(DTYPE[c["dtype"]])}


def _norm(x, kind, w, b, eps=1e-5):
    """(x normalised, its reciprocal deviation, the result)."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    rs = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = x * rs
    y = xh * w.float()
    return xh, rs, y + b.float() if b is not None else y


def _norm_back(dy, xh, rs, kind, w):
    """The gradients of a norm's input, weight and bias."""
    dxh = dy * w.float()
    dx = dxh - xh * (dxh * xh).mean(-1, keepdim=True)
    if kind == "layer":
        dx = dx - dxh.mean(-1, keepdim=True)
    return dx * rs, (dy * xh).sum(0), dy.sum(0)


def _plain_norm(s):
    c, dt, kind = s["c"], DTYPE[s["c"]["dtype"]], s["c"]["kind"]
    x, block = s["x"].float(), s["block"].float()
    n1 = block
    if c["post"]:
        bh, rs1, n1 = _norm(block, kind, s["post_weight"], s["post_bias"])
    gated = n1
    if c["gate"]:
        g = s["gate"].float().repeat_interleave(c["n"] // c["gate"], 0)
        gated = g * n1
    r = s["scale"] * x + gated
    rh, rs2, h = _norm(r, kind, s["pre_weight"], s["pre_bias"])
    out = {"r": r.to(dt), "h": h.to(dt)}
    if c["dir"] == "fwd":
        return out
    back, dpw, dpb = _norm_back(s["dh"].float(), rh, rs2, kind, s["pre_weight"])
    dr = s["dr"].float() + back
    out["dx"], out["dpre_weight"] = (s["scale"] * dr).to(dt), dpw.to(dt)
    if kind == "layer":
        out["dpre_bias"] = dpb.to(dt)
    dn1 = dr
    if c["gate"]:
        dn1 = dr * g
        out["dgate"] = (dr * n1).view(c["gate"], -1, c["d"]).sum(1).to(dt)
    if c["post"]:
        dn1, dqw, dqb = _norm_back(dn1, bh, rs1, kind, s["post_weight"])
        out["dpost_weight"] = dqw.to(dt)
        if kind == "layer":
            out["dpost_bias"] = dqb.to(dt)
    out["dblock"] = dn1.to(dt)
    return out


def _visible(c, mask):
    """Which keys each row sees: [b or 1, 1, t, s]."""
    t, S = c["t"], c["s"]
    i = torch.arange(S - t, S, device="cuda")[:, None]
    j = torch.arange(S, device="cuda")[None, :]
    see = j <= i
    if c["window"]:
        see = see & ((i - j < c["window"]) | (j < c["sinks"]))
    see = see[None, None]
    return see if mask is None else see & mask[:, None, None, :]


def _plain_attn(s):
    c, dt = s["c"], DTYPE[s["c"]["dtype"]]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if s["mask"] is not None:
        k, v = (x.masked_fill(~s["mask"][:, None, :, None], 0.0) for x in (k, v))
    kk, vv = (x.repeat_interleave(c["group"], 1) for x in (k, v))
    see = _visible(c, s["mask"])
    p = torch.matmul(q, kk.transpose(-1, -2).contiguous()).mul_(s["scale"]).masked_fill_(~see, NEG)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == NEG, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    out = {"out": torch.matmul(p, vv).to(dt)}
    if c["dir"] == "fwd":
        return out
    do = s["do"].float()
    shared = lambda x: x.view(c["b"], c["hk"], c["group"], c["s"], c["d"]).sum(2).to(dt)  # noqa: E731
    out["dv"] = shared(torch.matmul(p.transpose(-1, -2).contiguous(), do))
    ds = torch.matmul(do, vv.transpose(-1, -2).contiguous())
    ds = ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
    out["dq"] = torch.matmul(ds, kk).to(dt)
    out["dk"] = shared(torch.matmul(ds.transpose(-1, -2).contiguous(), q))
    return out


def _plain_dist(s):
    c, dt = s["c"], DTYPE[s["c"]["dtype"]]
    z, T, a = s["logits"].float(), c["temp"], c["alpha"]
    live = s["ids"] >= 0
    at = s["ids"].clamp_min(0)
    taught = live.any(-1, keepdim=True)
    t = (s["teacher"].float() / T).masked_fill(~live, NEG)
    tt = t - torch.where(taught, t.amax(-1, keepdim=True), 0.0)
    e = tt.exp()
    total = torch.where(taught, e.sum(-1, keepdim=True), 1.0)
    p = e / total
    zt = z / T
    top = zt.amax(-1, keepdim=True)
    ez = (zt - top).exp()
    sz = ez.sum(-1, keepdim=True)
    lse = top + sz.log()
    logq = zt.gather(1, at) - lse
    kd = T * T * torch.where(live, p * (torch.where(live, tt, 0.0) - total.log() - logq), 0.0).sum(-1)
    loss = a * kd
    if c["labels"]:
        named = s["labels"] >= 0
        lab = s["labels"].clamp_min(0)[:, None]
        top1 = z.amax(-1, keepdim=True)
        e1 = (z - top1).exp()
        s1 = e1.sum(-1, keepdim=True)
        ce = (top1 + s1.log() - z.gather(1, lab))[:, 0]
        loss = loss + (1 - a) * torch.where(named, ce, 0.0)
    if c["dir"] == "fwd":
        return {"loss": loss}
    w = s["drow"][:, None]
    dz = ez / sz * (w * a * T * taught)
    dz.scatter_add_(1, at, -torch.where(live, p, 0.0) * (w * a * T))
    if c["labels"]:
        wl = w * (1 - a) * named[:, None]
        dz += e1 / s1 * wl
        dz.scatter_add_(1, lab, -wl)
    return {"loss": loss, "dlogits": dz.to(dt)}


# ------------------------------------------------------------------ the framework's operators
def _own(s):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import stquant_lm as lm
    c = s["c"]
    if c["op"] == "emb":
        out = lm.embedding_forward(s["tokens"], s["weight"], scale=s["scale"], dtype=DTYPE[c["out"]])
        if c["dir"] == "fwd":
            return {"out": out}
        return {"out": out, "dweight": lm.embedding_backward(s["grad"], s["tokens"], c["vocab"], scale=s["scale"], padding_idx=s["padding"],
                                                              dtype=DTYPE[c["dtype"]])}
    if c["op"] == "norm":
        kw = dict(pre_bias=s["pre_bias"], post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"], residual_scale=s["scale"],
                  kind=c["kind"])
        r, h, stats = lm.norm_residual_forward(s["x"], s["block"], s["pre_weight"], eps=1e-5, **kw)
        out = {"r": r, "h": h}
        if c["dir"] == "train":
            grads = lm.norm_residual_backward(s["dr"], s["dh"], s["x"], s["block"], s["pre_weight"], stats, **kw)
            out.update({"d" + name: g for name, g in grads.items()})
        return out
    if c["op"] == "attn":
        kw = dict(window=c["window"], sinks=c["sinks"], scale=s["scale"], key_mask=s["mask"])
        o, lse = lm.attention_forward(s["q"], s["k"], s["v"], **kw)
        if c["dir"] == "fwd":
            return {"out": o}
        dq, dk, dv = lm.attention_backward(s["do"], s["q"], s["k"], s["v"], o, lse, **kw)
        return {"out": o, "dq": dq, "dk": dk, "dv": dv}
    kw = dict(labels=s["labels"], temperature=c["temp"], alpha=c["alpha"])
    if c["dir"] == "fused":
        loss, dz = lm.distill_loss_and_grad(s["logits"], s["teacher"], s["ids"], grad=s["drow"], **kw)
        return {"loss": loss, "dlogits": dz}
    loss, stats = lm.distill_loss_forward(s["logits"], s["teacher"], s["ids"], **kw)
    if c["dir"] == "fwd":
        return {"loss": loss}
    return {"loss": loss, "dlogits": lm.distill_loss_backward(s["drow"], s["logits"], s["teacher"], s["ids"], stats, **kw)}


def run(state):
    if own:
        return _own(state)
    return {"emb": _plain_emb, "norm": _plain_norm, "attn": _plain_attn, "dist": _plain_dist}[state["c"]["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def _pairs(c):
    """How many (row, key) pairs a head's rows see."""
    total = 0
    w, k0 = c["window"] or c["s"], c["sinks"] if c["window"] else 0
    for pad in _pads(c):
        # row at position p sees keys pad..p that lie in the window or among the first k0
        for lo, hi, f in _pieces(c["s"] - c["t"], c["s"], pad, w, k0):
            total += (hi - lo) * (f(lo) + f(hi - 1)) / 2
    return total / c["b"]


def _pieces(first, last, pad, w, k0):
    """[first, last) cut where the count of visible keys changes its slope, each piece with its (linear) count."""
    def count(p):
        own_window = max(0, p - max(pad, p - w + 1) + 1)
        return own_window + max(0, min(k0, p - w + 1) - pad)
    cuts = sorted({min(max(x, first), last) for x in (first, last, pad, pad + w, w - 1, w, w + k0, w - 1 + k0, pad + w - 1)})
    return [(a, b, count) for a, b in zip(cuts, cuts[1:]) if b > a]


def work(case):
    c, z = case, SIZE[case["dtype"]]
    train = c["dir"] != "fwd"
    if c["op"] == "emb":
        rows, o = min(c["n"], c["vocab"]), SIZE[c["out"]]
        by = rows * c["d"] * z + c["n"] * (8 + c["d"] * o)
        return {"bytes": by + train * (c["n"] * c["d"] * o + c["vocab"] * c["d"] * z), "flops": c["n"] * c["d"] * (1 + 2 * train)}
    if c["op"] == "norm":
        e = c["n"] * c["d"]
        # forward: x and the block read, r and h written; backward: both read again with dr and dh, dx and dblock written
        return {"bytes": e * z * (10 if train else 4), "flops": e * (8 + 30 * train + (6 + 10 * train) * c["post"])}
    if c["op"] == "attn":
        h = c["hk"] * c["group"]
        q, kv = c["b"] * h * c["t"] * c["d"] * z, 2 * c["b"] * c["hk"] * c["s"] * c["d"] * z
        # forward: q, k, v read, out written; backward: those, dout and out read, dq, dk, dv written
        return {"bytes": 2 * q + kv + train * (4 * q + 2 * kv), "flops": c["b"] * h * _pairs(c) * c["d"] * (14 if train else 4)}
    e = c["n"] * c["vocab"]
    # the logits read (twice where a later call makes the gradient) and their gradient written
    return {"bytes": e * z * {"fwd": 1, "fused": 2, "train": 3}[c["dir"]] + c["n"] * c["k"] * (8 + z), "flops": e * (6 if c["dir"] == "fwd" else 10)}


# ------------------------------------------------------------------ the same in 64 bits, by automatic differentiation
def _leaf(t):
    return None if t is None else t.double().detach().requires_grad_(True)


def _exact_emb(s):
    c = s["c"]
    # (a float32 scale, as the operators take it)
    scale = float(torch.tensor(s["scale"], dtype=torch.float32))
    out = s["weight"].double().index_select(0, s["tokens"]) * scale
    if c["dir"] == "fwd":
        return {"out": out}
    keep = torch.ones_like(s["tokens"], dtype=torch.bool) if s["padding"] is None else s["tokens"] != s["padding"]
    rows = torch.zeros(c["vocab"], c["d"], dtype=torch.float64, device="cuda")
    rows.index_put_((s["tokens"][keep],), s["grad"].double()[keep], accumulate=True)
    return {"out": out, "dweight": rows * scale}


def _exact_norm(s):
    c = s["c"]
    names = ("x", "block", "pre_weight", "pre_bias", "post_weight", "post_bias", "gate")
    v = {k: _leaf(s[k]) for k in names}

    def norm(y, w, b):
        if c["kind"] == "layer":
            var, mean = torch.var_mean(y, -1, unbiased=False, keepdim=True)
            y = (y - mean) / torch.sqrt(var + 1e-5)
        else:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-5)
        return torch.addcmul(b, y, w) if b is not None else y * w

    y = v["block"] if v["post_weight"] is None else norm(v["block"], v["post_weight"], v["post_bias"])
    if v["gate"] is not None:
        y = (y.view(c["gate"], -1, c["d"]) * v["gate"][:, None]).view(c["n"], c["d"])
    r = y + v["x"] * float(torch.tensor(s["scale"], dtype=torch.float32))
    h = norm(r, v["pre_weight"], v["pre_bias"])
    out = {"r": r.detach(), "h": h.detach()}
    if c["dir"] == "train":
        have = [k for k in names if v[k] is not None]
        grads = torch.autograd.grad([r, h], [v[k] for k in have], [s["dr"].double(), s["dh"].double()])
        out.update({"d" + k: g for k, g in zip(have, grads)})
    return out


def _exact_attn(s):
    c = s["c"]
    train = c["dir"] == "train"
    h = c["hk"] * c["group"]
    out = {"out": torch.zeros(c["b"], h, c["t"], c["d"], dtype=torch.float64, device="cuda")}
    if train:
        out["dq"] = torch.zeros_like(out["out"])
        out["dk"], out["dv"] = (torch.zeros(c["b"], c["hk"], c["s"], c["d"], dtype=torch.float64, device="cuda") for _ in range(2))
    pos = torch.arange(c["s"] - c["t"], c["s"], device="cuda")
    key = torch.arange(c["s"], device="cuda")
    gap = pos[:, None] - key[None, :]
    hidden = gap < 0
    if c["window"]:
        hidden |= (gap >= c["window"]) & (key >= c["sinks"])[None, :]
    for b in range(c["b"]):
        gone = hidden if s["mask"] is None else hidden | ~s["mask"][b][None, :]
        empty = gone.all(-1, keepdim=True)
        gone = gone & ~empty          # an empty row: any finite weights, dropped below
        for i in range(h):
            q, k, v = _leaf(s["q"][b, i]), _leaf(s["k"][b, i // c["group"]]), _leaf(s["v"][b, i // c["group"]])
            w = torch.softmax((q @ k.t().contiguous() * s["scale"]).masked_fill(gone, NEG), -1)
            o = (w @ v).masked_fill(empty, 0.0)
            out["out"][b, i] = o.detach()
            if train:
                dq, dk, dv = torch.autograd.grad(o, [q, k, v], s["do"][b, i].double())
                out["dq"][b, i] = dq
                out["dk"][b, i // c["group"]] += dk
                out["dv"][b, i // c["group"]] += dv
    return out


def _exact_dist(s):
    c, T, a = s["c"], s["c"]["temp"], s["c"]["alpha"]
    loss = torch.zeros(c["n"], dtype=torch.float64, device="cuda")
    dz = torch.zeros(c["n"], c["vocab"], dtype=torch.float64, device="cuda") if c["dir"] != "fwd" else None
    rows = max(1, (1 << 27) // c["vocab"])
    for r in range(0, c["n"], rows):
        at = slice(r, min(r + rows, c["n"]))
        z = _leaf(s["logits"][at])
        ids, there = s["ids"][at], s["ids"][at] >= 0
        some = there.any(-1)
        teach = torch.where(there, s["teacher"][at].double() / T, torch.full((), -1e300, dtype=torch.float64, device="cuda"))
        logp = torch.log_softmax(teach, -1)
        p = torch.where(there, logp.exp(), 0.0)
        logq = torch.log_softmax(z / T, -1).gather(1, ids.clamp_min(0))
        row = a * T * T * torch.where(there, p * (torch.where(there, logp, 0.0) - torch.where(there, logq, 0.0)), 0.0).sum(-1)
        row = torch.where(some, row, 0.0)
        if c["labels"]:
            row = row + (1.0 - a) * torch.nn.functional.cross_entropy(z, s["labels"][at], ignore_index=-100, reduction="none")
        loss[at] = row.detach()
        if dz is not None:
            dz[at] = torch.autograd.grad(row, z, s["drow"][at].double())[0]
    return {"loss": loss} if dz is None else {"loss": loss, "dlogits": dz}


def exact(case, seed):
    s = prepare(case, seed)
    return {"emb": _exact_emb, "norm": _exact_norm, "attn": _exact_attn, "dist": _exact_dist}[case["op"]](s)
