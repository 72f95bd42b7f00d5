"""Routing, expert products, their combination and clipping in 64 bits (plain torch), and the inputs their tests share.

Bounds: a sum of K products of 16-bit values is formed in fp32 with at most K + 1 roundings of 2^-24, each of at most the
sum of the terms' magnitudes, before its one rounding to the result's type."""
import torch

import lm_reference as ref

EPS32 = 2.0 ** -24


def sorted_slots(ids, experts):
    """(rows, places, offsets) by a stable sort on the host."""
    flat = ids.detach().cpu().long().view(-1)
    key = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    rows = torch.sort(key, stable=True)[1]
    places = torch.empty_like(rows)
    places[rows] = torch.arange(rows.numel())
    offsets = torch.tensor([int((key < e).sum()) for e in range(experts + 1)])
    return rows, places.view(ids.shape), offsets


def choices(g, n, experts, k, absent=0.0, skew=False, dtype=torch.int32):
    """[n, k] different experts a token, some slots of none (-1, or an id behind the last expert)."""
    score = torch.rand(n, experts, device="cuda", generator=g)
    if skew:
        score = score * torch.linspace(1.0, 0.05, experts, device="cuda")
    ids = torch.topk(score, k, dim=1)[1].to(dtype)
    if absent:
        u = torch.rand(n, k, device="cuda", generator=g)
        ids[u < absent / 2] = -1
        ids[u > 1 - absent / 2] = experts
    return ids


def product(x, weight, ids, gather, dy=None):
    """y, dx, dweight of the sorted slots, each with the sum of magnitudes that went into it."""
    experts, k = weight.shape[0], ids.shape[-1]
    rows, _, offsets = sorted_slots(ids, experts)
    rows, off = rows.to(x.device), offsets.tolist()
    width = x.shape[-1]
    xs = x.reshape(-1, width).double()
    src = rows // k if gather else torch.arange(rows.numel(), device=x.device)
    y, ym = (torch.zeros(rows.numel(), weight.shape[1], dtype=torch.float64, device=x.device) for _ in range(2))
    out = {"y": (y, ym)}
    if dy is not None:
        dx, dxm = (torch.zeros_like(xs) for _ in range(2))
        dw, dwm = (torch.zeros(weight.shape, dtype=torch.float64, device=x.device) for _ in range(2))
        out.update(dx=(dx, dxm), dweight=(dw, dwm))
    for e in range(experts):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        w, xe = weight[e].double(), xs[src[a:b]]
        y[a:b], ym[a:b] = xe @ w.t(), xe.abs() @ w.abs().t()
        if dy is not None:
            g = dy[a:b].double()
            dx.index_add_(0, src[a:b], g @ w)
            dxm.index_add_(0, src[a:b], g.abs() @ w.abs())
            dw[e], dwm[e] = g.t() @ xe, g.abs().t() @ xe.abs()
    if dy is not None:
        out["dx"] = tuple(t.view(x.shape) for t in out["dx"])
    return out


def check_product(got, want, terms):
    """Each result against its 64-bit value: terms[name] products were added."""
    for name, (w, mag) in want.items():
        ref.within(name, got[name], w, (terms[name] + 1) * EPS32 * mag)


def combine(y, weights, ids, experts):
    """out of the sorted rows y."""
    _, places, offsets = sorted_slots(ids, experts)
    places, live = places.to(y.device), int(offsets[-1])
    there = places < live
    w = torch.ones(places.shape, dtype=torch.float64, device=y.device) if weights is None else weights.double()
    rows = torch.where(there[..., None], y.double()[places], torch.zeros((), dtype=torch.float64, device=y.device))
    return (torch.where(there, w, torch.zeros_like(w))[..., None] * rows).sum(-2)


def route(logits, k, renormalize):
    """(weights, ids, load) of [n, experts] logits; differentiable in 64 bits."""
    z = logits.double()
    open_ = logits.detach() > ref.NEG
    some = open_.any(-1, keepdim=True)
    top = torch.where(some, z.detach().amax(-1, keepdim=True), torch.zeros_like(z[:, :1]))
    e = torch.where(open_, (torch.where(open_, z, torch.zeros_like(z)) - top).exp(), torch.zeros_like(z))
    p = e / torch.where(some, e.sum(-1, keepdim=True), torch.ones_like(z[:, :1]))
    order = torch.sort(logits.detach().double(), dim=-1, descending=True, stable=True)[1][:, :k]
    there = open_.gather(1, order)
    w = torch.where(there, p.gather(1, order), torch.zeros_like(p[:, :k]))
    if renormalize:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(some, total, torch.ones_like(total))
    return w, torch.where(there, order, torch.full_like(order, -1)), p.sum(0)


def clip(grads, max_norm, norm=None):
    """(norm, the scaled gradients) in 64 bits."""
    if norm is None:
        norm = sum((float((g.double() ** 2).sum()) for g in grads), 0.0) ** 0.5
    c = min(1.0, max_norm / (norm + 1e-6)) if norm == norm else norm
    return norm, [g.double() * c for g in grads]
