"""The distillation loss over all its temperatures and over logits of any size, against 64 bits."""
import pytest
import torch

import lm_reference as ref
import stquant_lm as lm

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def both(z, t, ids, lab, temp, alpha):
    """(loss, gradient) of the two calls that read the logits once, which must be those of the pair of calls."""
    w = torch.ones(z.shape[0], device="cuda")
    kw = dict(labels=lab, temperature=temp, alpha=alpha)
    loss, dz = lm.distill_loss_and_grad(z, t, ids, grad=w, **kw)
    l2, stats = lm.distill_loss_forward(z, t, ids, **kw)
    d2 = lm.distill_loss_backward(w, z, t, ids, stats, **kw)
    leaf = z.double().detach().requires_grad_(True)
    want = ref.distill(leaf, t, ids, lab, temp, alpha)
    return (loss, l2), (dz, d2), want.detach(), torch.autograd.grad(want.sum(), leaf)[0]


@pytest.mark.parametrize("temp", [1e-15, 1e-12, 3e-10, 1e-7, 1e-4, 0.03])
@pytest.mark.parametrize("v", [900, 60000, 120000])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_small_temperatures(temp, v, dtype):
    """Whole logits: their differences are exact, so that at small temperatures every weight is 0, 1 or shared among
    equal ones, and the loss a difference of logits times T.  Exponents of up to 30 / T carry 2^-22 of themselves: they
    round to weights of 0 all the same."""
    g = ref.gen(v)
    n, k = 5, 9
    z = torch.randint(-20, 11, (n, v), device="cuda", generator=g).to(dtype)
    z[:, 17] = 11.0
    z[1, 500] = 11.0                              # two largest
    ids = torch.stack([torch.randperm(v, device="cuda", generator=g)[:k] for _ in range(n)])
    ids[0, 0] = 17
    t = torch.stack([torch.randperm(k, device="cuda", generator=g) for _ in range(n)]).to(dtype)
    lab = torch.randint(0, v, (n,), device="cuda", generator=g)
    for alpha, labels in ((1.0, None), (0.6, lab)):
        loss, dz, wl, wd = both(z, t, ids, labels, temp, alpha)
        for x in loss:
            ref.within("loss", x, wl, 2.0 ** -20 * (wl.abs() + 32 * (1 - alpha) + 32 * temp))
        for x in dz:
            ref.within("dlogits", x, wd, 2.0 ** -16 * (wd.abs() + alpha * temp + (1 - alpha) * torch.softmax(z.double(), -1)))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("temp", [0.5, 1.0, 2.0, 3.0])
@pytest.mark.parametrize("v", [300, 60000])
def test_rows_of_the_lowest_and_of_huge_logits(dtype, temp, v):
    """A row that a mask of the type's lowest value leaves nothing of is uniform; logits of the largest size have
    differences like any others."""
    n, k = 6, 4
    low = torch.finfo(dtype).min
    big = torch.finfo(dtype).max
    z = torch.zeros(n, v, dtype=dtype, device="cuda")
    z[0], z[1], z[2] = low, big, low
    z[2, 7] = big                                 # certain
    z[3, 100:] = low                              # 100 left
    z[4] = low / 2
    z[5, 50:] = float("-inf")
    ids = torch.arange(k, device="cuda").expand(n, k).contiguous()
    ids[2] = torch.tensor([7, -1, -1, -1])
    t = torch.zeros(n, k, dtype=dtype, device="cuda")
    t[1], t[3] = low, big                         # alike, at either end
    lab = torch.full((n,), 3, device="cuda")
    lab[2] = 7
    loss, dz, wl, wd = both(z, t, ids, lab, temp, 0.5)
    assert bool(torch.isfinite(wl).all())
    for x in loss:
        ref.within("loss", x, wl, 2.0 ** -18 * (wl.abs() + 12 * temp * temp + 12))
    # (hidden logits weigh exactly nothing; at the entries and the label terms of up to T and 1 cancel)
    terms = (wd != 0).double().scatter(1, torch.where(ids < 0, ids[:, :1], ids), 1.0).scatter(1, lab[:, None], 1.0)
    for x in dz:
        ref.within("dlogits", x, wd, 2.0 ** -18 * (wd.abs() + temp + 1) * terms)


@pytest.mark.parametrize("temp", [0.5, 1.0, 2.0, 3.0, 4.0, 50.0])
@pytest.mark.parametrize("e", [12, 20, 24, 26, 27, 28, 29, 30, 31, 32, 36, 60, 120])
def test_neighbours_of_a_large_logit(e, temp):
    """fp32 logits a few spacings below 2^e: exponents whose rounded offset is up to 64, which a weight of T = 4 carries
    four times: 2^-24 * 64 * 4 of each weight, and four times that allowed; what weighs less than 2^-31 may be 0."""
    n, v, k = 4, 260, 5
    top, ulp = 2.0 ** e, 2.0 ** (e - 24)
    g = ref.gen(e)
    z = torch.full((n, v), -top, device="cuda")
    z[:, :40] = top - ulp * torch.randint(0, 24, (n, 40), device="cuda", generator=g).float()
    z[:, 3] = top
    ids = torch.stack([torch.randperm(40, device="cuda", generator=g)[:k] for _ in range(n)])
    t = ref.randn(g, n, k)
    lab = torch.randint(0, 40, (n,), device="cuda", generator=g)
    loss, dz, wl, wd = both(z, t, ids, lab, temp, 0.5)
    q = torch.softmax(z.double() / temp, -1) * temp + torch.softmax(z.double(), -1)
    at = torch.zeros_like(q).scatter(1, ids, temp).scatter_add(1, lab[:, None], torch.ones(n, 1, dtype=torch.float64, device="cuda"))
    for x in loss:
        ref.within("loss", x, wl, 2.0 ** -14 * (temp * temp + 1) + 2.0 ** -18 * (temp + 1) * 24 * ulp)
    for x in dz:
        ref.within("dlogits", x, wd, 2.0 ** -14 * (q + at) + 2.0 ** -31 * (temp + 1) * (z > 0))


@pytest.mark.parametrize("n", [3, 600])
@pytest.mark.parametrize("v", [5, 33, 300, 2100, 9000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_nothing_behind_a_row_is_written(n, v, dtype):
    """Rows so far apart that whatever a workgroup's last threads would write behind their row lies in the gap."""
    stride = (1 << 18) // (2 if dtype == BF16 else 4) if n < 600 else 1 << 15
    g = ref.gen(v)
    z = torch.full((n, stride), 3.0, dtype=dtype, device="cuda")
    z[:, :v] = ref.randn(g, n, v, dtype=dtype)
    ids = torch.zeros(n, 1, dtype=torch.int64, device="cuda")
    t = torch.zeros(n, 1, dtype=dtype, device="cuda")
    out = torch.full((n, stride), 7.0, dtype=dtype, device="cuda")
    lm.distill_loss_and_grad(z[:, :v], t, ids, grad=1.0, out=out[:, :v])
    assert bool((out[:, v:] == 7).all())
    _, stats = lm.distill_loss_forward(z[:, :v], t, ids)
    lm.distill_loss_backward(1.0, z[:, :v], t, ids, stats, out=out[:, :v])
    assert bool((out[:, v:] == 7).all())


@pytest.mark.parametrize("v", [1000, 12000, 50257, 60000])
@pytest.mark.parametrize("temp,top", [(1e-9, 11.0), (1e-4, 11.0), (2.0, 3e38), (3.0, -3e38), (4.0, 1e9)])
def test_many_rows_of_steep_logits(v, temp, top):
    """The instances for more than 512 rows, in place: rows of a value and of ones far below it."""
    n, k = 520, 3
    z = torch.full((n, v), top, device="cuda").to(BF16)
    z[:, 5:] = -z[:, 5:].abs() / 2 if top > 0 else float("-inf")
    ids = torch.arange(k, device="cuda").expand(n, k).contiguous()
    t = torch.zeros(n, k, dtype=BF16, device="cuda")
    w = torch.full((n,), 1.0, device="cuda")
    loss, dz = lm.distill_loss_and_grad(z, t, ids, grad=w, temperature=temp, out=z)
    # uniform over 5, the teacher over 3 of them
    want = torch.zeros(n, v, dtype=torch.float64, device="cuda")
    want[:, :5] = temp / 5
    want[:, :3] -= temp / 3
    ref.within("loss", loss, torch.full((n,), temp * temp * 0.5108256237659907, dtype=torch.float64, device="cuda"), 2.0 ** -16 * temp * temp)
    ref.within("dlogits", dz, want, 2.0 ** -16 * temp * (want != 0))
