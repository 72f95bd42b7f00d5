"""The transformer operators' definitions in 64 bits (plain torch, any device), and what their tests share.

``U[dtype]`` is the largest relative error of one rounding to a type; ``F32`` allows for the fp32 work
between roundings: sums of up to 2^6 terms a lane and the steps of a reduction stay below 2^6 roundings of
2^-24, and exponentials of arguments up to 64 below 64 * 2^-24, so 2^-17 of the magnitudes that went into a
value covers both."""
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}     # below: absolute rounding
F32 = 2.0 ** -17
NEG = float("-inf")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, std=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(*shape, device="cuda", generator=g) * std + mean).to(dtype)


def within(name, got, want, bound):
    """|got - want| <= bound + one rounding to got's type, element by element; NaN and infinities alike."""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    g, w = got.double(), want.double()
    fine = torch.isfinite(w)
    assert torch.equal(torch.isfinite(g), fine), f"{name}: other values are finite"
    assert torch.equal(torch.isnan(g), torch.isnan(w)) and torch.equal(g[torch.isinf(w)], w[torch.isinf(w)]), name
    lim = bound + U[got.dtype] * w.abs() + TINY[got.dtype]
    over = (g - w).abs() - lim
    over = torch.where(fine, over, torch.full_like(over, -1.0))
    if over.numel() and float(over.max()) > 0:
        at = int(over.argmax())
        raise AssertionError(f"{name}: element {at} is {g.reshape(-1)[at]} for {w.reshape(-1)[at]}, "
                             f"allowed {lim.expand_as(w).reshape(-1)[at]}; {int((over > 0).sum())} of {over.numel()} over")


def differences(f, args, which, direction, step):
    """The derivative of the sum f(*args) along ``direction`` of args[which], by central differences in 64 bits."""
    a, b = list(args), list(args)
    a[which] = args[which].double() + step * direction
    b[which] = args[which].double() - step * direction
    return (f(*a) - f(*b)) / (2 * step)


# ---------------------------------------------------------------- embedding
def embedding_grad(grad, tokens, vocab, scale=1.0, padding=None):
    """(the gradient, the sum of magnitudes that went into it)."""
    g, t = grad.double().reshape(-1, grad.shape[-1]), tokens.reshape(-1).long()
    keep = (t >= 0) & (t < vocab)
    if padding is not None:
        keep &= t != padding
    out, mag = (torch.zeros(vocab, g.shape[1], dtype=torch.float64, device=g.device) for _ in range(2))
    out.index_put_((t[keep],), g[keep] * scale, accumulate=True)
    mag.index_put_((t[keep],), g[keep].abs() * abs(scale), accumulate=True)
    return out, mag


# ---------------------------------------------------------------- residual norms
def norm(y, w, b, kind, eps):
    if kind == "layer":
        y = y - y.mean(-1, keepdim=True)
    y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w
    return y if b is None else y + b


def norm_residual(x, block, pre_weight, pre_bias, post_weight, post_bias, gate, scale, eps, kind):
    d = x.shape[-1]
    y = block if post_weight is None else norm(block, post_weight, post_bias, kind, eps)
    if gate is not None:
        g = gate.reshape(-1, d)
        y = (y.reshape(g.shape[0], -1, d) * g[:, None]).reshape(x.shape)
    r = scale * x + y
    return r, norm(r, pre_weight, pre_bias, kind, eps)


# ---------------------------------------------------------------- attention
def visible(t, s, window, sinks, key_mask, b, device):
    i = torch.arange(s - t, s, device=device)[:, None]
    j = torch.arange(s, device=device)[None, :]
    see = (j <= i) & ((i - j < window) | (j < sinks)) if window else j <= i
    see = see.expand(b, t, s)
    return see if key_mask is None else see & key_mask.bool()[:, None, :]


def attention(q, k, v, window=0, sinks=0, scale=None, key_mask=None):
    """(out, lse, weights) in 64 bits; q [b, h, t, d], k and v [b, hk, s, d]."""
    b, h, t, d = q.shape
    hk, s = k.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    if key_mask is not None:        # what a masked key holds does not matter
        k, v = (torch.where(key_mask.bool()[:, None, :, None], x, torch.zeros((), dtype=x.dtype, device=x.device)) for x in (k, v))
    kk, vv = (x.double().repeat_interleave(h // hk, 1) for x in (k, v))
    see = visible(t, s, window, sinks, key_mask, b, q.device)[:, None]
    scores = (q.double() @ kk.transpose(-1, -2).contiguous() * scale).masked_fill(~see, NEG)
    lse = torch.logsumexp(scores, -1)
    p = torch.where(see, (scores - torch.where(lse == NEG, torch.zeros_like(lse), lse)[..., None]).exp(), torch.zeros_like(scores))
    return p @ vv, lse, p


def attention_with_bounds(q, k, v, do, **kw):
    """out, dq, dk, dv in 64 bits, each with what the roundings on the way may put into it: the weights and their
    gradients rounded once to the type (u), delta formed from the rounded out."""
    b, h, t, d = q.shape
    hk, s = k.shape[1:3]
    scale = d ** -0.5 if kw.get("scale") is None else kw["scale"]
    mask = kw.get("key_mask")
    if mask is not None:
        k, v = (torch.where(mask.bool()[:, None, :, None], x, torch.zeros((), dtype=x.dtype, device=x.device)) for x in (k, v))
    u = U[q.dtype] + F32
    o, lse, p = attention(q, k, v, **kw)
    kk, vv = (x.double().repeat_interleave(h // hk, 1) for x in (k, v))
    g, qq = do.double(), q.double()
    dp = g @ vv.transpose(-1, -2).contiguous()
    delta = (g * o).sum(-1, keepdim=True)
    ds = p * (dp - delta) * scale
    # delta's error (u of |do| |o|), and fp32's in dp and p
    e_ds = p * scale * (u * (g.abs() * o.abs()).sum(-1, keepdim=True)
                        + 4 * F32 * (g.abs() @ vv.abs().transpose(-1, -2).contiguous() + (g * o).abs().sum(-1, keepdim=True))) + u * ds.abs()
    tr = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    shared = lambda x: x.reshape(b, hk, h // hk, s, d).sum(2)  # noqa: E731
    return {
        "out": (o, u * (p @ vv.abs()) + F32 * o.abs()),
        "lse": (lse, None),
        "dq": (ds @ kk, e_ds @ kk.abs()),
        "dk": (shared(tr(ds) @ qq), shared(tr(e_ds) @ qq.abs())),
        "dv": (shared(tr(p) @ g), u * shared(tr(p) @ g.abs())),
    }


# ---------------------------------------------------------------- distillation
def distill(logits, teacher, ids, labels, temp, alpha):
    """The loss of each row in 64 bits."""
    z, v = logits.double(), logits.shape[-1]
    there = (ids >= 0) & (ids < v)
    at = torch.where(there, ids, torch.zeros_like(ids)).long()
    t = torch.where(there, teacher.double() / temp, torch.full((), NEG, dtype=torch.float64, device=z.device))
    some = there.any(-1) & (t.amax(-1) > NEG) if t.shape[-1] else torch.zeros(z.shape[0], dtype=torch.bool, device=z.device)
    loss = torch.zeros(z.shape[0], dtype=torch.float64, device=z.device)
    if bool(some.any()):
        zs, ts, as_, th = z[some], t[some], at[some], there[some]
        lp = torch.log_softmax(ts, -1)
        p = lp.exp()
        lq = torch.log_softmax(zs / temp, -1).gather(1, as_)
        use = th & (p > 0)
        kd = torch.where(use, p * (torch.where(use, lp, torch.zeros_like(lp)) - torch.where(use, lq, torch.zeros_like(lq))), torch.zeros_like(p)).sum(-1)
        loss = loss.index_put((some.nonzero()[:, 0],), alpha * temp * temp * kd)
    if labels is not None and alpha != 1.0:
        named = (labels >= 0) & (labels < v)
        if bool(named.any()):
            ce = torch.nn.functional.cross_entropy(z[named], labels[named].long(), reduction="none")
            loss = loss.index_put((named.nonzero()[:, 0],), (1 - alpha) * ce, accumulate=True)
    return loss
