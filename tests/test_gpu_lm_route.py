"""Routing, plans and the combination of experts' rows against 64 bits: every spread of experts over lanes, ties, closed
experts, rows without any, NaN, strides, many slots.

Tolerances: probabilities are exponentials of differences of up to 16 here, sums of up to 512 of them and a division: below
2^-17 of their magnitude (lm_reference.F32).  The load adds n of them in fp32: n + 1 roundings at most of its size."""
import pytest
import torch

import lm_expert_reference as er
import lm_reference as ref
import stquant_lm as lm

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def check(logits, k, renormalize, seed=5, dweights=True, dload=True):
    n, e = logits.shape
    g = ref.gen(seed)
    dw = ref.randn(g, n, k) if dweights else None
    dl = ref.randn(g, e) if dload else None
    w, ids, load = lm.route_forward(logits, k, renormalize=renormalize)
    dz = lm.route_backward(dw, dl, logits, w, ids, renormalize=renormalize)
    z = logits.double().detach().requires_grad_(True)
    ww, wi, wl = er.route(z, k, renormalize)
    assert torch.equal(ids.long(), wi)
    ref.within("weights", w, ww.detach(), 2 * ref.F32 * ww.detach())
    ref.within("load", load, wl.detach(), (ref.F32 + n * er.EPS32) * wl.detach() + 1e-30)
    total = sum((d.double() * x).sum() for d, x in ((dw, ww), (dl, wl)) if d is not None)
    want = torch.autograd.grad(total, z)[0]
    # p or w times differences of gradients: each term's magnitude carries 2^-17
    p = torch.softmax(torch.where(logits.double() > ref.NEG, logits.double(), torch.full_like(z, -1e300)), -1).detach()
    size = (dl.abs().max().double() if dload else 0.0) * 2 + (dw.abs().double().amax(-1, keepdim=True) if dweights else 0.0)
    share = torch.zeros_like(p)
    share.scatter_add_(1, wi.clamp_min(0), ww.detach() * (wi >= 0))
    ref.within("dlogits", dz, want, 8 * ref.F32 * (p + share) * size + 1e-30)
    return w, ids, load, dz


@pytest.mark.parametrize("experts,k", [(1, 1), (2, 2), (7, 3), (8, 8), (9, 4), (16, 2), (31, 5), (33, 33), (64, 6), (65, 64), (128, 8), (200, 7), (256, 8), (511, 9), (512, 64)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("renormalize", [False, True])
def test_against_64_bits(experts, k, dtype, renormalize):
    g = ref.gen(experts)
    z = ref.randn(g, 77, experts, std=2.0, dtype=dtype)
    if experts > 4:
        z[torch.rand(z.shape, device="cuda", generator=g) < 0.2] = ref.NEG
        z[3] = ref.NEG
        z[5, 1:] = ref.NEG
    check(z, k, renormalize)


@pytest.mark.parametrize("n", [0, 1, 3, 31, 1025, 20000])
def test_rows(n):
    z = ref.randn(ref.gen(n), n, 60, std=3.0, dtype=BF16)
    if n:
        check(z, 4, False)
    else:
        w, ids, load = lm.route_forward(z, 4)
        assert w.shape == ids.shape == (0, 4) and torch.equal(load, torch.zeros(60, device="cuda"))
        assert lm.route_backward(w, load, z, w, ids).shape == (0, 60)


def test_equal_logits_go_to_the_lowest_expert():
    z = torch.zeros(5, 130, device="cuda")
    z[1] = -0.0
    z[2, 64:] = 1.0
    z[3, ::3] = 2.0
    z[4, 7], z[4, 3] = 0.0, -0.0
    _, ids, _ = lm.route_forward(z, 4)
    assert ids.tolist() == [[0, 1, 2, 3], [0, 1, 2, 3], [64, 65, 66, 67], [0, 3, 6, 9], [0, 1, 2, 3]]
    check(ref.randn(ref.gen(1), 400, 64, std=0.3).round(decimals=1), 8, True)


def test_lowest_and_largest_logits():
    """The type's lowest value is a logit like any other, -inf none at all."""
    for dtype in (F32, BF16, F16):
        low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
        z = torch.full((4, 12), low, device="cuda", dtype=dtype)
        z[1, 4], z[2, :6], z[3, 5] = high, ref.NEG, 0.0
        w, ids, load = lm.route_forward(z, 3, renormalize=True)
        assert ids.tolist() == [[0, 1, 2], [4, 0, 1], [6, 7, 8], [5, 0, 1]]
        want = torch.tensor([[1 / 3] * 3, [1.0, 0, 0], [1 / 3] * 3, [1.0, 0, 0]], device="cuda")
        assert float((w - want).abs().max()) <= 2.0 ** -22 and bool(torch.isfinite(load).all())


def test_nan_and_infinite_rows():
    z = ref.randn(ref.gen(2), 4, 20)
    z[1, 7], z[2, 3] = float("nan"), float("inf")
    w, ids, load = lm.route_forward(z, 3)
    assert bool(torch.isnan(w[1]).all()) and bool(torch.isnan(w[2]).all()) and bool(torch.isfinite(w[0]).all()) and bool(torch.isfinite(w[3]).all())
    assert int(ids[1, 0]) == 7 and int(ids[2, 0]) == 3 and bool((ids >= 0).all()) and bool((ids < 20).all())
    assert bool(torch.isnan(load).all())
    dz = lm.route_backward(torch.ones_like(w), None, z, w, ids)
    assert bool(torch.isnan(dz[1]).all()) and bool(torch.isfinite(dz[0]).all()) and bool(torch.isfinite(dz[3]).all())


def test_missing_gradients_and_leading_dimensions():
    z = ref.randn(ref.gen(3), 50, 24)
    check(z, 2, True, dweights=False)
    check(z, 2, False, dload=False)
    w, ids, load = lm.route_forward(z.view(5, 10, 24), 2)
    flat = lm.route_forward(z, 2)
    assert w.shape == (5, 10, 2) and all(torch.equal(a.reshape(b.shape), b) for a, b in zip((w, ids, load), flat))


def test_strided_logits():
    wide = ref.randn(ref.gen(4), 90, 80, dtype=BF16)
    for z in (wide[:, 3:43], wide[::2, 1:41], wide[:, ::2], wide[:1].expand(90, 80)[:, :40]):
        check(z, 3, False)


def test_autograd_and_differences():
    g = ref.gen(6)
    z = ref.randn(g, 9, 12).requires_grad_(True)
    dw, dl = ref.randn(g, 9, 3), ref.randn(g, 12)
    for renormalize in (False, True):
        w, ids, load = lm.route(z, 3, renormalize=renormalize)
        assert not ids.requires_grad
        got = torch.autograd.grad((w * dw).sum() + (load * dl).sum(), z)[0]
        f = lambda x: (lambda r: (r[0] * dw.double()).sum() + (r[2] * dl.double()).sum())(er.route(x, 3, renormalize))  # noqa: E731
        step = ref.randn(g, 9, 12).double()
        want = ref.differences(f, [z.detach()], 0, step, 1e-6)
        assert abs(float((got.double() * step).sum() - want)) <= 1e-4 * float((got.double() * step).abs().sum())
    with pytest.raises(RuntimeError):
        w, _, _ = lm.route(z, 3)
        torch.autograd.grad(torch.autograd.grad(w.sum(), z, create_graph=True)[0].sum(), z)


@pytest.mark.parametrize("n,k", [(0, 1), (0, 2), (1, 1), (5, 3), (64, 1), (1000, 2), (4096, 1), (4097, 1), (30000, 4), (400000, 3)])
@pytest.mark.parametrize("experts", [1, 2, 8, 60, 512])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_plan(n, k, experts, dtype):
    ids = torch.randint(-1, experts + 1, (n, k), device="cuda", generator=ref.gen(n + experts)).to(dtype)
    if dtype == torch.int64 and n:
        ids[0, 0] = 1 << 40
    if n > 100000 and experts > 60:
        ids[: n // 2] = 3                       # one long run
    plan = lm.expert_plan(ids, experts)
    rows, places, offsets = er.sorted_slots(ids, experts)
    assert torch.equal(plan.rows.cpu().long(), rows) and torch.equal(plan.places.cpu().long(), places) and torch.equal(plan.offsets.cpu().long(), offsets)


def test_plan_of_strided_ids():
    ids = torch.randint(0, 9, (50, 6), device="cuda", generator=ref.gen(1), dtype=torch.int32)[:, ::2]
    plan = lm.expert_plan(ids, 9)
    assert torch.equal(plan.rows.cpu().long(), er.sorted_slots(ids, 9)[0])


@pytest.mark.parametrize("n,k,dim", [(1, 1, 1), (3, 2, 8), (7, 5, 100), (130, 4, 768), (33, 8, 1025), (5, 64, 24), (20000, 2, 16), (9, 3, 11008)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("weighted", [True, False])
def test_combine(n, k, dim, dtype, weighted):
    g, experts = ref.gen(n + dim), 70
    ids = er.choices(g, n, experts, k, absent=0.2)
    plan = lm.expert_plan(ids, experts)
    y = ref.randn(g, n * k, dim, dtype=dtype)
    live = int(plan.offsets[-1])
    y[live:] = float("nan")                     # what rows of no expert hold does not matter
    w = torch.rand(n, k, device="cuda", generator=g) if weighted else None
    do = ref.randn(g, n, dim, dtype=dtype)
    out = lm.expert_combine_forward(y, w, plan)
    dy, dw = lm.expert_combine_backward(do, y, w, plan)
    y64 = torch.where(torch.arange(n * k, device="cuda")[:, None] < live, y.double(), 0.0).requires_grad_(True)
    w64 = (torch.ones(n, k, device="cuda") if w is None else w).double().requires_grad_(True)
    want = er.combine(y64, w64, ids, experts)
    gy, gw = torch.autograd.grad(want, [y64, w64], do.double())
    mag = er.combine(y64.detach().abs(), w64.detach(), ids, experts)
    ref.within("out", out, want.detach(), (k + 1) * er.EPS32 * mag)
    ref.within("dy", dy, gy, er.EPS32 * gy.abs())
    assert not bool(dy[live:].any())
    if weighted:
        mags = torch.autograd.grad(er.combine(y64.detach().abs(), w64, ids, experts), w64, do.double().abs())[0]
        ref.within("dweights", dw, gw, (dim + 1) * er.EPS32 * mags)
    else:
        assert dw is None
    assert lm.expert_combine_backward(do, y, w, plan, weight_grads=False)[1] is None


def test_combine_strides():
    g = ref.gen(8)
    ids = er.choices(g, 40, 10, 2)
    plan = lm.expert_plan(ids.view(5, 8, 2), 10)
    wide = ref.randn(g, 80, 65, dtype=BF16)
    w = torch.rand(5, 16, 2, device="cuda", generator=g)[:, ::2]
    for y in (wide[:, 1:33], wide[:, :64:2], wide[:1].expand(80, 65)[:, :24]):
        do = ref.randn(g, y.shape[1], 5, 8, dtype=BF16).permute(1, 2, 0)
        dense = [t.clone(memory_format=torch.contiguous_format) for t in (y, w, do)]
        assert torch.equal(lm.expert_combine_forward(y, w, plan), lm.expert_combine_forward(dense[0], dense[1], plan))
        for a, b in zip(lm.expert_combine_backward(do, y, w, plan), lm.expert_combine_backward(dense[2], dense[0], dense[1], plan)):
            assert torch.equal(a, b)


def test_combine_of_no_tokens():
    plan = lm.expert_plan(torch.zeros(0, 2, dtype=torch.int32, device="cuda"), 4)
    y = torch.zeros(0, 16, device="cuda")
    assert lm.expert_combine_forward(y, None, plan).shape == (0, 16)
