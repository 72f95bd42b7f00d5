"""Routing, expert products, their combination and clipping together, as ``distill_pretrain.py`` uses them: one step of a
sparse decoder against the same model in plain fp32 torch, training with the 4-bit optimizer, graphs and streams."""
import copy
import math

import pytest
import torch

import distill_pretrain as dp
import lm_expert_reference as er
import lm_reference as ref
import stquant_lm as lm

pytestmark = pytest.mark.gpu
SMALL = dict(vocab=515, n_embd=128, n_layer=2, n_head=4, n_kv=2, window=24, sinks=2, experts=6, top_experts=2, expert_width=200)


def plain(model, tokens, choices):
    """The model's logits and load term in fp32 torch operations, its experts chosen as given (a choice between two nearly
    equal logits may fall either way)."""
    rms = lambda x, w: x * (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w  # noqa: E731
    b, t = tokens.shape
    d, hd, n = model.wte.shape[1], model.dim, tokens.numel()
    x = model.wte[tokens] * math.sqrt(d)
    h = rms(x, model.first)
    see = ref.visible(t, t, model.window, model.sinks, None, b, tokens.device)[:, None]
    uneven = 0.0
    for i in range(2 * model.n_layer):
        if i % 2:
            flat, ids = h.reshape(n, d), choices[i // 2].view(n, -1).long()
            p = torch.softmax(flat @ model.router[i // 2].t(), -1)
            w = p.gather(1, ids)
            w = w / w.sum(-1, keepdim=True)
            y = torch.zeros_like(flat)
            for e in range(model.experts):
                u = torch.nn.functional.gelu(flat @ model.up[i // 2][e].t(), approximate="tanh") @ model.down[i // 2][e].t()
                y = y + ((ids == e) * w).sum(-1, keepdim=True) * u
            share = torch.bincount(ids.view(-1), minlength=model.experts) / ids.numel()
            uneven = uneven + model.experts * (share * p.mean(0)).sum() / model.n_layer
            y = y.view(b, t, d)
        else:
            kv = model.n_kv * hd
            q, k, v = (z.view(b, t, -1, hd).transpose(1, 2) for z in (h @ model.qkv[i // 2].t()).split([d, kv, kv], -1))
            k, v = (z.repeat_interleave(model.n_head // model.n_kv, 1) for z in (k, v))
            p = torch.softmax((q @ k.transpose(-1, -2).contiguous() * hd ** -0.5).masked_fill(~see, ref.NEG), -1)
            y = (p @ v).transpose(1, 2).reshape(b, t, d) @ model.proj[i // 2].t()
        x = x + model.gate[i] * rms(y, model.post[i])
        h = rms(x, model.pre[i])
    return h @ model.wte.t(), uneven


def test_one_step_against_plain_torch(monkeypatch):
    model, teacher = dp.Decoder(seed=1, **SMALL), dp.Decoder(seed=2, **SMALL)
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() >= 2:
                p.mul_(3.0)            # scores and logits of a trained model's size
    tokens = torch.randint(0, 515, (3, 77), device="cuda", generator=ref.gen(0))
    targets = dp.teach(teacher, tokens, 16)
    choices, route = [], lm.route
    monkeypatch.setattr(lm, "route", lambda *a, **k: (choices.append(route(*a, **k)) or choices[-1]))
    loss = dp.step_loss(model, tokens, targets, temperature=2.0, alpha=0.6, balance=0.5)
    uneven = float(model.uneven)
    got = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad(set_to_none=True)
    labels = torch.full_like(tokens, -100)
    labels[:, :-1] = tokens[:, 1:]
    logits, even = plain(model, tokens, [c[1] for c in choices])
    want = ref.distill(logits.view(-1, 515), targets[0].view(-1, 16), targets[1].view(-1, 16), labels.view(-1), 2.0, 0.6).mean()
    (want + 0.5 * even).backward()
    assert abs(float(loss) - float(want.detach())) <= 0.01 * abs(float(want.detach()))
    assert abs(uneven - float(even.detach())) <= 0.01 * float(even.detach())
    # about 15 roundings of activations and as many of their gradients to bfloat16 (each 2^-9 of its array in the
    # mean) lie between a weight and the loss: 2^-9 sqrt(30) is 1.1 %, and five times that is allowed
    for n, p in model.named_parameters():
        off = float((got[n] - p.grad).norm() / p.grad.norm())
        assert off <= 0.055, (n, off)


def test_a_step_leaves_no_graph_behind():
    """A model that still held the step's graph could not be copied, and a backward pass of its weights not be captured."""
    model, teacher = dp.Decoder(seed=1, **SMALL), dp.Decoder(seed=2, **SMALL)
    tokens = torch.randint(0, 515, (2, 30), device="cuda", generator=ref.gen(0))
    dp.step_loss(model, tokens, dp.teach(teacher, tokens, 16), temperature=2.0, alpha=0.6)
    assert model.uneven.grad_fn is None and not model.uneven.requires_grad and float(model.uneven) > 0.0
    twin = copy.deepcopy(model)
    assert all(torch.equal(a, b) for a, b in zip(twin.parameters(), model.parameters()))


def test_training_with_the_low_bit_optimizer_and_clipping():
    """It runs, every expert's parameters move, and each step's gradients keep to the norm."""
    norms, clip = [], lm.clip_grads

    def spy(grads, most):
        norm = clip(grads, most)
        norms.append((float(norm), sum(float(g.double().square().sum()) for g in grads) ** 0.5))
        return norm
    lm.clip_grads = spy
    try:
        res = dp.train(steps=12, warmup=1, batch=4, seq_len=64, lr=2e-3, k=16, vocab_used=64, max_grad_norm=0.05, **SMALL)
    finally:
        lm.clip_grads = clip
    assert len(norms) == 13 and all(math.isfinite(x) for x in res["Losses"])
    for before, after in norms:
        assert before > 0.05 and abs(after - 0.05 * before / (before + 1e-6)) <= 1e-5 * 0.05


def test_every_expert_learns(monkeypatch):
    """Each expert's matrices and each router have a gradient in every step, and all of them differ from where they began."""
    models, made, clip = [], dp.Decoder, lm.clip_grads

    def spy(grads, most):
        grads = list(grads)
        for g in grads:
            if g.dim() == 3:
                assert bool((g.flatten(1).abs().amax(1) > 0).all())
        assert sum(g.dim() == 3 for g in grads) == 4
        return clip(grads, most)
    monkeypatch.setattr(dp, "Decoder", lambda **k: (models.append(made(**k)) or models[-1]))
    monkeypatch.setattr(lm, "clip_grads", spy)
    dp.train(steps=3, warmup=1, batch=4, seq_len=64, lr=2e-3, k=16, vocab_used=64, max_grad_norm=0.05, **SMALL)
    model, before = models[0], made(seed=42, **SMALL)
    for name in ("up", "down", "router"):
        for a, b in zip(getattr(model, name), getattr(before, name)):
            assert bool(((a - b).flatten(1).abs().amax(1) > 0).all()), name


def layer(x, logits, up, down, k=2):
    w, ids, load = lm.route(logits, k, renormalize=True)
    plan = lm.expert_plan(ids, up.shape[0])
    y = lm.expert_product(torch.relu(lm.expert_product(x, up, plan, gather=True)), down, plan)
    return lm.expert_combine(y, w, plan), load


def operands(n, experts, d, width, seed=0):
    g = ref.gen(seed)
    x, logits = ref.randn(g, n, d, dtype=torch.bfloat16), ref.randn(g, n, experts, std=2.0)
    return x, logits, ref.randn(g, experts, width, d, std=d ** -0.5, dtype=torch.bfloat16), ref.randn(g, experts, d, width, std=width ** -0.5, dtype=torch.bfloat16)


@pytest.mark.parametrize("n", [1, 24, 1400, 6000])
def test_a_layer_with_its_gradients(n):
    """Against 64 bits.  Three results are rounded to bfloat16 on the way forward and as many backward, each by up to 2^-8 of
    its own; six of those, of the largest value in an array, bound the difference."""
    ops = [t.requires_grad_(True) for t in operands(n, 5, 64, 96)]
    out, load = layer(*ops)
    do = ref.randn(ref.gen(9), n, 64, dtype=torch.bfloat16)
    got = torch.autograd.grad([out, load], ops, [do, torch.ones_like(load)])
    x, logits, up, down = wide = [t.detach().double().requires_grad_(True) for t in ops]
    w, ids, lo = er.route(logits, 2, True)
    want = torch.zeros(n, 64, dtype=torch.float64, device="cuda")
    for e in range(5):
        u = torch.relu(x @ up[e].t()) @ down[e].t()
        want = want + ((ids == e) * w).sum(-1, keepdim=True) * u
    ref_grads = torch.autograd.grad([want, lo], wide, [do.double(), torch.ones_like(lo)])
    for name, a, b in zip(("out", "x", "logits", "up", "down"), (out, *got), (want, *ref_grads)):
        assert float((a.double() - b).abs().max()) <= 6 * ref.U[torch.bfloat16] * float(b.abs().max()), name


def test_captured_and_replayed():
    """Forward, backward and clipping in one graph, replayed over new inputs between other work."""
    x, logits, up, down = operands(700, 6, 64, 96)
    do = ref.randn(ref.gen(2), 700, 64, dtype=torch.bfloat16)

    def step():
        w, ids, load = lm.route_forward(logits, 2)
        plan = lm.expert_plan(ids, 6)
        u = lm.expert_product_forward(x, up, plan, gather=True)
        y = lm.expert_product_forward(u, down, plan)
        out = lm.expert_combine_forward(y, w, plan)
        dy, dw = lm.expert_combine_backward(do, y, w, plan)
        du, ddown = lm.expert_product_backward(dy, u, down, plan)
        dx, dup = lm.expert_product_backward(du, x, up, plan, gather=True)
        dz = lm.route_backward(dw, load, logits, w, ids)
        norm = lm.clip_grads([dup, ddown, dz], 0.5)
        return out, load, dx, dup, ddown, dz, norm, plan.rows, plan.offsets
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(4):
        for t, new in zip((x, logits, up, down), operands(700, 6, 64, 96, seed=seed)):
            t.copy_(new)
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), seed


def test_another_stream():
    x, logits, up, down = operands(900, 6, 64, 96)
    want = [t.clone() for t in layer(x, logits, up, down)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(x, logits, up, down)
        norm = lm.grad_norm([x, up])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and float(norm) == float(lm.grad_norm([x, up]))


def test_two_streams_at_once():
    """Calls on two streams share nothing: each has its workspace."""
    ops = [operands(n, 6, 64, 96, seed=n) for n in (1300, 5000)]
    want = [[t.clone() for t in layer(*o)] for o in ops]
    streams = [torch.cuda.Stream() for _ in ops]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((*layer(*ops[i]), lm.grad_norm(ops[i])))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert torch.equal(g[0], want[i][0]) and torch.equal(g[1], want[i][1]) and float(g[2]) == float(got[i][0][2])


def test_norms_on_two_streams_at_once():
    """Against norms formed beforehand, one at a time."""
    lists = [[ref.randn(ref.gen(i), n + 7 * i, dtype=d) for n in (5, 40_000, 300_001) for d in (torch.float32, torch.bfloat16)] for i in range(2)]
    want = [er.clip(g, 1.0)[0] for g in lists]
    streams = [torch.cuda.Stream() for _ in lists]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                out = [torch.empty_like(g) for g in lists[i]]
                got[i].append((lm.clip_grads(lists[i], 1.0, out=out), lm.grad_norm(lists[i]), out))
    torch.cuda.synchronize()
    for i in range(2):
        for norm, again, out in got[i]:
            assert abs(float(norm) - want[i]) <= want[i] * (2.0 ** -24 + 2.0 ** -40) and float(again) == float(norm)
            for o, g in zip(out, er.clip(lists[i], 1.0)[1]):
                ref.within("gradient", o, g, 2.0 ** -23 * g.abs())
