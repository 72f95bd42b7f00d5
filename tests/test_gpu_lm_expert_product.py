"""The experts' products, forward and backward, against 64 bits: runs from no row to many, tiles that are not full, gathered
and sorted rows, slots of no expert, strides, both types.  The tolerance counts the roundings of fp32 sums
(lm_expert_reference)."""
import pytest
import torch

import lm_expert_reference as er
import lm_reference as ref
import stquant_lm as lm

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def operands(n, experts, k, din, dout, dtype, gather, seed=None, absent=0.0, skew=False):
    g = ref.gen(n + din + dout if seed is None else seed)
    ids = er.choices(g, n, experts, k, absent=absent, skew=skew)
    x = ref.randn(g, n if gather else n * k, din, dtype=dtype)
    w = ref.randn(g, experts, dout, din, std=din ** -0.5, dtype=dtype)
    dy = ref.randn(g, n * k, dout, dtype=dtype)
    return ids, x, w, dy


def check(ids, x, w, dy, gather, dtype=None):
    experts, dout, din = w.shape
    plan = lm.expert_plan(ids, experts)
    y = lm.expert_product_forward(x, w, plan, gather=gather)
    dx, dw = lm.expert_product_backward(dy, x, w, plan, gather=gather, dtype=dtype)
    assert dw.dtype == (dtype or w.dtype)
    most = int((plan.offsets[1:] - plan.offsets[:-1]).max()) if ids.numel() else 0
    er.check_product(dict(y=y, dx=dx, dweight=dw), er.product(x, w, ids, gather, dy), dict(y=din, dx=dout + ids.shape[-1], dweight=most))
    return y, dx, dw


# tokens, experts, choices, in, out
SIZES = [(1, 1, 1, 8, 8), (1, 8, 2, 64, 40), (3, 4, 2, 16, 136), (17, 5, 1, 72, 24), (40, 64, 2, 128, 264), (130, 3, 2, 264, 72), (257, 8, 2, 200, 128),
         (500, 60, 4, 64, 200), (1000, 2, 1, 96, 520), (700, 1, 1, 328, 392), (2000, 16, 3, 40, 48)]


@pytest.mark.parametrize("n,experts,k,din,dout", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("gather", [False, True])
def test_against_64_bits(n, experts, k, din, dout, dtype, gather):
    ids, x, w, dy = operands(n, experts, k, din, dout, dtype, gather)
    check(ids, x, w, dy, gather)


# more tiles than workgroups, of both sizes, with tails of rows, columns and k; many rows an expert, one or none of them
LARGE = [(4000, 4, 2, 1032, 4104), (4000, 4, 2, 4104, 264), (3001, 2, 2, 4200, 4360), (13000, 3, 1, 2056, 1096), (3001, 2, 1, 72, 3080), (2500, 60, 4, 136, 4104), (9000, 1, 1, 520, 264), (700, 64, 1, 96, 2056), (513, 1, 1, 64, 64),
         (4100, 8, 1, 128, 192)]


@pytest.mark.parametrize("n,experts,k,din,dout", LARGE)
@pytest.mark.parametrize("dtype,gather,skew", [(BF16, True, False), (BF16, False, True), (F16, True, True), (F16, False, False)])
def test_many_tiles(n, experts, k, din, dout, dtype, gather, skew):
    ids, x, w, dy = operands(n, experts, k, din, dout, dtype, gather, skew=skew, absent=0.1 if skew else 0.0)
    check(ids, x, w, dy, gather)


def test_one_expert_takes_all():
    """Every other expert's run is empty; the one that is not lies first, last or between."""
    for n in (20, 1500, 9000):
        for e in (0, 5, 15):
            ids, x, w, dy = operands(n, 16, 1, 80, 136, BF16, True)
            ids.fill_(e)
            y, dx, dw = check(ids, x, w, dy, True)
            assert not bool(dw[[i for i in range(16) if i != e]].any())


@pytest.mark.parametrize("experts", [63, 64, 65, 130, 512])
def test_many_experts(experts):
    """The search for a tile goes 64 experts at a time."""
    for n in (experts // 3, 40 * experts):
        ids, x, w, dy = operands(n, experts, 1, 24, 40, BF16, False, absent=0.1)
        check(ids, x, w, dy, False)


def test_few_rows_and_more_tiles_than_workgroups():
    ids, x, w, dy = operands(256, 64, 2, 8, 131080, BF16, True)
    plan = lm.expert_plan(ids, 64)
    y = lm.expert_product_forward(x, w, plan, gather=True)
    er.check_product(dict(y=y), er.product(x, w, ids, True), dict(y=8))


@pytest.mark.parametrize("n,experts,din,dout", [(30, 8, 136, 200), (900, 6, 136, 520), (5000, 4, 264, 520)])
def test_the_same_call_gives_the_same_bits(n, experts, din, dout):
    ids, x, w, dy = operands(n, experts, 2, din, dout, BF16, True)
    plan = lm.expert_plan(ids, experts)
    run = lambda: (lm.expert_product_forward(x, w, plan, gather=True), *lm.expert_product_backward(dy, x, w, plan, gather=True))  # noqa: E731
    first = run()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("skew", [False, True])
def test_slots_of_no_expert(gather, skew):
    """Their rows come out as zeros and add nothing, whatever they hold."""
    for n, experts in ((60, 20), (900, 7), (2100, 2)):
        ids, x, w, dy = operands(n, experts, 2, 88, 160, BF16, gather, absent=0.3, skew=skew)
        live = int(lm.expert_plan(ids, experts).offsets[-1])
        dy[live:] = float("nan")
        if gather:
            x[((ids < 0) | (ids >= experts)).all(-1)] = float("nan")
        else:
            x[live:] = float("inf")
        clean = [torch.where(torch.isfinite(t), t, torch.zeros_like(t)) for t in (x, dy)]
        plan = lm.expert_plan(ids, experts)
        y = lm.expert_product_forward(x, w, plan, gather=gather)
        dx, dw = lm.expert_product_backward(dy, x, w, plan, gather=gather)
        assert not bool(y[live:].any())
        want = check(ids, clean[0], w, clean[1], gather)
        assert all(torch.equal(a, b) for a, b in zip((y, dx, dw), want))


def test_no_slot_has_an_expert():
    ids = torch.full((50, 2), -1, device="cuda", dtype=torch.int32)
    _, x, w, dy = operands(50, 6, 2, 24, 32, BF16, True)
    y, dx, dw = check(ids, x, w, dy, True)
    assert not bool(y.any()) and not bool(dx.any()) and not bool(dw.any())


@pytest.mark.parametrize("gather", [False, True])
def test_no_tokens(gather):
    ids = torch.zeros(0, 2, device="cuda", dtype=torch.int32)
    _, _, w, _ = operands(1, 6, 2, 24, 32, BF16, True)
    x, dy = torch.zeros(0, 24, device="cuda", dtype=BF16), torch.zeros(0, 32, device="cuda", dtype=BF16)
    plan = lm.expert_plan(ids, 6)
    assert lm.expert_product_forward(x, w, plan, gather=gather).shape == (0, 32)
    dx, dw = lm.expert_product_backward(dy, x, w, plan, gather=gather)
    assert dx.shape == (0, 24) and not bool(dw.any())


@pytest.mark.parametrize("n,experts,k,din,dout", [(300, 5, 2, 136, 200), (20, 8, 2, 64, 96)])
def test_fp32_weight_gradients(n, experts, k, din, dout):
    ids, x, w, dy = operands(n, experts, k, din, dout, BF16, True, skew=True)
    check(ids, x, w, dy, True, dtype=torch.float32)


@pytest.mark.parametrize("n,experts,k,din,dout", [(4000, 4, 2, 1032, 4104), (3001, 2, 2, 4200, 4360), (700, 64, 1, 264, 520), (6000, 130, 1, 256, 256)])
@pytest.mark.parametrize("dtype,gather,skew", [(BF16, True, True), (F16, False, False)])
def test_fp32_weight_gradients_in_large_tiles(n, experts, k, din, dout, dtype, gather, skew):
    """More tiles than workgroups, full ones and cut ones, experts of no row among them."""
    ids, x, w, dy = operands(n, experts, k, din, dout, dtype, gather, skew=skew, absent=0.1 if skew else 0.0)
    ids[ids == experts - 1] = 0
    check(ids, x, w, dy, gather, dtype=torch.float32)


def test_parts_of_the_backward_pass():
    ids, x, w, dy = operands(200, 6, 2, 72, 104, F16, True)
    plan = lm.expert_plan(ids, 6)
    dx, dw = lm.expert_product_backward(dy, x, w, plan, gather=True)
    a, b = lm.expert_product_backward(dy, x, w, plan, gather=True, weights=False)
    c, d = lm.expert_product_backward(dy, x, w, plan, gather=True, inputs=False)
    assert torch.equal(a, dx) and b is None and c is None and torch.equal(d, dw)


@pytest.mark.parametrize("n", [9, 400])
def test_strides(n):
    """Views whose rows begin on 16 bytes are read as they are, others copied: the same bits."""
    ids, x, w, dy = operands(n, 6, 2, 72, 104, BF16, True)
    plan = lm.expert_plan(ids, 6)
    want = (lm.expert_product_forward(x, w, plan, gather=True), *lm.expert_product_backward(dy, x, w, plan, gather=True))

    def inside(t, off, pad):
        wide = torch.full((*t.shape[:-1], t.shape[-1] + pad), float("nan"), dtype=t.dtype, device="cuda")
        wide[..., off:off + t.shape[-1]] = t
        return wide[..., off:off + t.shape[-1]]
    for off, pad in ((8, 16), (1, 5)):
        for xs, ws, ds in ((inside(x, off, pad), w, dy), (x, inside(w, off, pad), dy), (x, w, inside(dy, off, pad)),
                           (x.t().contiguous().t(), w.transpose(1, 2).contiguous().transpose(1, 2), dy.t().contiguous().t())):
            got = (lm.expert_product_forward(xs, ws, plan, gather=True), *lm.expert_product_backward(ds, xs, ws, plan, gather=True))
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    three = (lm.expert_product_forward(x.view(n // 1, 1, 72), w, plan._replace(places=plan.places.view(n, 1, 2)), gather=True),
             *lm.expert_product_backward(dy, x.view(n, 1, 72), w, plan._replace(places=plan.places.view(n, 1, 2)), gather=True))
    assert all(torch.equal(a.view(b.shape), b) for a, b in zip(three, want))


def test_an_expert_far_behind_in_memory():
    """Expert matrices more than 2^31 bytes apart."""
    ids, x, w, dy = operands(40, 2, 1, 64, 64, BF16, True)
    far = torch.zeros((1 << 30) + (1 << 13), dtype=BF16, device="cuda")
    view = far.as_strided(w.shape, ((1 << 30) + 64, 64, 1))
    view.copy_(w)
    plan = lm.expert_plan(ids, 2)
    assert torch.equal(lm.expert_product_forward(x, view, plan, gather=True), lm.expert_product_forward(x, w, plan, gather=True))
    assert torch.equal(lm.expert_product_backward(dy, x, view, plan, gather=True)[0], lm.expert_product_backward(dy, x, w, plan, gather=True)[0])


def test_autograd_and_differences():
    ids, x, w, dy = operands(23, 4, 2, 24, 32, BF16, True)
    plan = lm.expert_plan(ids, 4)
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = lm.expert_product(x, w, plan, gather=True)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    want = lm.expert_product_backward(dy, x.detach(), w.detach(), plan, gather=True)
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])
    g = ref.gen(77)
    for which, grad in ((0, dx), (1, dw)):
        step = ref.randn(g, *grad.shape).double()
        f = lambda a, b: (er.product(a, b, ids, True)["y"][0] * dy.double()).sum()  # noqa: E731
        diff = ref.differences(f, [x.detach(), w.detach()], which, step, 1e-4)
        # each gradient is rounded once, by up to 2^-8 of it, and independently: four deviations of the sum of those
        size = float(((grad.double() * step) ** 2).sum().sqrt())
        assert abs(float((grad.double() * step).sum()) - float(diff)) <= 4 * ref.U[BF16] * size + 1e-6
    only = torch.autograd.grad(lm.expert_product(x.detach(), w, plan, gather=True), w, dy)[0]
    assert torch.equal(only, dw)


def test_plans_that_do_not_fit_are_refused():
    ids, x, w, dy = operands(23, 4, 2, 24, 32, BF16, True)
    plan = lm.expert_plan(ids, 5)
    with pytest.raises(RuntimeError, match="the plan is for 5 experts, weight has 4"):
        lm.expert_product_forward(x, w, plan, gather=True)
    plan = lm.expert_plan(ids, 4)
    with pytest.raises(RuntimeError, match="x must be"):
        lm.expert_product_forward(x, w, plan)
    with pytest.raises(RuntimeError, match="dy must be"):
        lm.expert_product_backward(dy[:5], x, w, plan, gather=True)
    with pytest.raises(RuntimeError, match="dweight must be"):
        lm.expert_product_backward(dy, x, w, plan, gather=True, dtype=F16)
    with pytest.raises(RuntimeError, match="multiples of 8"):
        lm.expert_product_forward(x[:, :20].contiguous(), w[..., :20].contiguous(), plan, gather=True)
