"""The distillation loss and its gradient against 64 bits: types, vocabularies of every path (rows in registers and
rows read again), odd widths and strides, absent entries, repeated ids, labels, masked logits, empty rows.

Tolerances: an exponential of an argument of size x carries 2^-22 (1 + x) (the argument's and the function's fp32
errors), a sum of them no more; every gradient element is rounded once to its type."""
import pytest
import torch

import lm_reference as ref
import stquant_lm as lm

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def inputs(seed, n, v, k, dtype, labels=True, std=2.5):
    g = ref.gen(seed)
    z = ref.randn(g, n, v, std=std, dtype=dtype)
    ids = torch.randint(0, v, (n, k), device="cuda", generator=g)         # repeats among them where k is not small
    t = ref.randn(g, n, k, std=3.0, dtype=dtype)
    lab = torch.randint(0, v, (n,), device="cuda", generator=g) if labels else None
    return z, t, ids, lab, torch.rand(n, device="cuda", generator=g) + 0.1


def reference(z, t, ids, lab, temp, alpha, w):
    leaf = z.double().detach().requires_grad_(True)
    loss = ref.distill(leaf, t, ids, lab, temp, alpha)
    if not loss.requires_grad:
        return loss, torch.zeros_like(leaf)
    return loss.detach(), torch.autograd.grad((loss * w.double()).sum(), leaf)[0]


def bounds(z, temp, alpha, w, t):
    """What fp32 may put into the loss and the gradient: relative to the distributions' own sizes."""
    zz = torch.where(torch.isfinite(z.double()), z.double(), torch.zeros((), dtype=torch.float64, device=z.device))
    span = (zz.amax(-1) - zz.amin(-1)) / min(temp, 1.0) + 20
    if t.shape[-1]:
        span = span + 2 * t.double().abs().amax(-1) / temp
    e = 2.0 ** -22 * (1 + span)
    q = torch.softmax(z.double() / temp, -1) * temp * alpha + torch.softmax(z.double(), -1) * (1 - alpha)
    return e * (temp * temp * span + span), e[:, None] * w.double()[:, None] * q, e * w.double() * (alpha * temp + 1)


def check(z, t, ids, lab, w, temp=1.0, alpha=1.0, out=None):
    kw = dict(labels=lab, temperature=temp, alpha=alpha)
    want_loss, want = reference(z, t, ids, lab, temp, alpha, w)
    lb, db, point = bounds(z, temp, alpha, w, t)
    # at the row's entries and label the gradient is a difference of two terms of up to alpha T + 1
    at = torch.zeros_like(want)
    v = z.shape[1]
    if t.shape[1]:
        inside = (ids >= 0) & (ids < v)
        at.scatter_(1, torch.where(inside, ids, torch.zeros_like(ids)).long(), 1.0)
    if lab is not None:
        at.scatter_(1, lab.clamp(0, v - 1).long()[:, None], 1.0)
    db = torch.nan_to_num(db) + at * point[:, None]
    loss, stats = lm.distill_loss_forward(z, t, ids, **kw)
    ref.within("loss", loss, want_loss, lb)
    two = lm.distill_loss_backward(w, z, t, ids, stats, **kw)
    ref.within("dlogits", two, want, db)
    l1, one = lm.distill_loss_and_grad(z, t, ids, grad=w, out=out, **kw)
    ref.within("loss", l1, want_loss, lb)
    ref.within("dlogits", one, want, db)
    return loss, one


@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (3, 5, 3), (2, 300, 40), (5, 1000, 1), (4, 4099, 64), (3, 32000, 8), (6, 50257, 100), (2, 70001, 1024), (2, 150001, 16), (2, 300007, 5)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("temp,alpha", [(1.0, 1.0), (2.0, 0.7)])
def test_against_64_bits(n, v, k, dtype, temp, alpha):
    z, t, ids, lab, w = inputs(n + v, n, v, k, dtype)
    check(z, t, ids, lab if alpha < 1 else None, w, temp, alpha)


@pytest.mark.parametrize("alpha,labels", [(0.0, True), (0.5, True), (1.0, True), (0.5, False), (0.0, False)])
def test_mixtures(alpha, labels):
    z, t, ids, lab, w = inputs(1, 9, 700, 12, F32, labels)
    loss, _ = check(z, t, ids, lab, w, 3.0, alpha)
    if alpha == 0.0 and not labels:
        assert not bool(loss.any())


def test_absent_entries_and_labels():
    z, t, ids, lab, w = inputs(2, 8, 500, 6, BF16)
    ids[0, 3:], ids[1], ids[2, 0], ids[3, 1] = -1, -1, 500, 2 ** 40
    lab[1], lab[4], lab[5] = -100, 500, -1
    ids[4] = -7
    z[1], z[4] = float("nan"), float("inf")          # rows with neither entry nor label may hold anything
    loss, dz = check(torch.where(torch.isfinite(z), z, torch.zeros_like(z)), t, ids, lab, w, 2.0, 0.6)
    l2, d2 = lm.distill_loss_and_grad(z, t, ids, grad=w, labels=lab, temperature=2.0, alpha=0.6)
    assert torch.equal(l2, loss) and torch.equal(d2, dz) and not bool(l2[[1, 4]].any()) and not bool(d2[[1, 4]].any())
    stats = lm.distill_loss_forward(z, t, ids, labels=lab, temperature=2.0, alpha=0.6)[1]
    assert not bool(lm.distill_loss_backward(w, z, t, ids, stats, labels=lab, temperature=2.0, alpha=0.6)[[1, 4]].any())


def test_repeated_ids_and_a_label_among_them():
    z, t, ids, lab, w = inputs(3, 4, 90, 7, F32)
    ids[:, 1:5] = ids[:, :1]
    lab[:2] = ids[:2, 0]
    check(z, t, ids, lab, w, 1.5, 0.4)


def test_masked_logits():
    """-inf and the type's lowest value among the student's logits; -inf among the teacher's."""
    for dtype in (F32, BF16, F16):
        z, t, ids, lab, w = inputs(4, 6, 1003, 9, dtype)
        z[:, 500:700] = float("-inf")
        z[:, 700:800] = torch.finfo(dtype).min
        ids, lab = ids % 500, lab % 500
        t[0, 4:], t[1] = float("-inf"), float("-inf")
        check(z, t, ids, lab, w, 2.0, 0.5)
    # a teacher weight where the student's is zero: an infinite loss, a finite gradient
    ids[2, 0] = 600
    loss, dz = lm.distill_loss_and_grad(z, t, ids, grad=w, labels=lab, temperature=2.0, alpha=0.5)
    assert torch.isposinf(loss[2]) and bool(torch.isfinite(dz).all())


def test_nan_logits_stay_in_their_row():
    z, t, ids, lab, w = inputs(5, 4, 333, 5, F32)
    z[1, 7] = float("nan")
    loss, dz = lm.distill_loss_and_grad(z, t, ids, grad=w, labels=lab, alpha=0.5)
    assert bool(loss[1].isnan()) and bool(dz[1].isnan().any()) and not bool(dz[[0, 2, 3]].isnan().any())


@pytest.mark.parametrize("v,stride,shift,oshift", [(1001, 1001, 0, 0), (1000, 1007, 3, 3), (1000, 1003, 1, 2), (50257, 50304, 5, 5), (33, 33, 1, 0)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_at_any_offset(v, stride, shift, oshift, dtype):
    n = 5
    z, t, ids, lab, w = inputs(v, n, v, 11, dtype)
    buf, obuf = (torch.full((n * stride + s,), 7.0, dtype=dtype, device="cuda") for s in (shift, oshift))
    zv, out = buf[shift:].view(n, stride)[:, :v], obuf[oshift:].view(n, stride)[:, :v]
    zv.copy_(z)
    check(zv, t, ids, lab, w, 2.0, 0.5, out=out)
    assert bool((obuf[:oshift] == 7).all()) and bool((obuf[oshift:].view(n, stride)[:, v:] == 7).all())


@pytest.mark.parametrize("v", [37, 4001, 50257, 200003])
def test_in_place(v):
    z, t, ids, lab, w = inputs(v, 3, v, 20, BF16)
    kw = dict(labels=lab, temperature=2.0, alpha=0.5)
    loss, dz = lm.distill_loss_and_grad(z, t, ids, grad=w, **kw)
    _, stats = lm.distill_loss_forward(z, t, ids, **kw)
    z1, z2 = z.clone(), z.clone()
    l1, d1 = lm.distill_loss_and_grad(z1, t, ids, grad=w, out=z1, **kw)
    assert d1.data_ptr() == z1.data_ptr() and torch.equal(z1, dz) and torch.equal(l1, loss)
    lm.distill_loss_backward(w, z2, t, ids, stats, out=z2, **kw)
    assert torch.equal(z2, lm.distill_loss_backward(w, z, t, ids, stats, **kw))


def test_shapes_types_and_weights():
    z, t, ids, lab, w = inputs(6, 12, 260, 5, BF16)
    kw = dict(temperature=2.0, alpha=0.5)
    loss, dz = lm.distill_loss_and_grad(z, t, ids, grad=w, labels=lab, **kw)
    l2, d2 = lm.distill_loss_and_grad(z.view(3, 4, 260), t.float().view(3, 4, 5), ids.int().view(3, 4, 5), grad=w.view(3, 4), labels=lab.int().view(3, 4), **kw)
    assert torch.equal(l2.view(-1), loss) and torch.equal(d2.view(12, 260), dz)
    a = lm.distill_loss_and_grad(z, t, ids, grad=0.25, labels=lab, **kw)[1]
    assert torch.equal(a, lm.distill_loss_and_grad(z, t, ids, grad=torch.full((12,), 0.25, device="cuda"), labels=lab, **kw)[1])
    none = lm.distill_loss_and_grad(z, t[:, :0], ids[:, :0], grad=w, labels=lab, **kw)
    assert torch.allclose(none[0], 0.5 * torch.nn.functional.cross_entropy(z.float(), lab, reduction="none"), rtol=1e-5)
    e = lm.distill_loss_and_grad(z[:0], t[:0], ids[:0], grad=w[:0], labels=lab[:0], **kw)
    assert e[0].shape == (0,) and e[1].shape == (0, 260)


def test_autograd_and_differences():
    z, t, ids, lab, w = inputs(7, 10, 130, 6, F32)
    lab[3], ids[4] = -100, -1
    leaf = z.clone().requires_grad_(True)
    (lm.distill_loss(leaf, t, ids, labels=lab, temperature=2.0, alpha=0.6) * w).sum().backward()
    d = ref.randn(ref.gen(2), 10, 130).double()
    num = ref.differences(lambda x: (ref.distill(x, t, ids, lab, 2.0, 0.6) * w.double()).sum(), [z], 0, d, 1e-5)
    got = (leaf.grad.double() * d).sum()
    # 130 elements a row, each within 2^-22 * 40 of terms of up to w (alpha T + 1) = 2.5
    assert abs(float(num) - float(got)) <= 2.0 ** -22 * 40 * 2.5 * float(d.abs().sum()) + 1e-7
    leaf2 = z.clone().requires_grad_(True)
    lm.distill_loss(leaf2, t, ids, labels=lab, temperature=2.0, alpha=0.6).mean().backward()
    assert torch.allclose(leaf2.grad, lm.distill_loss_and_grad(z, t, ids, grad=0.1, labels=lab, temperature=2.0, alpha=0.6)[1], atol=1e-7)
